// Python bindings of packed causal attention and of the position bias.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "longctx_args.h"

extern "C" void dlb_packed_attn_fwd(const PaFwd* p, const PaBias* bias,
                                    int width, hipStream_t stream);
extern "C" void dlb_packed_attn_bwd_q(const PaBwd* p, const PaBias* bias,
                                      int width, hipStream_t stream);
extern "C" void dlb_packed_attn_bwd_kv(const PaBwd* p, const PaBias* bias,
                                       int width, void* dtable,
                                       int dtable_bf16, hipStream_t stream);
extern "C" void dlb_relbias_fwd(const void* table, void* out, const RbArgs* a,
                                int size, hipStream_t stream);
extern "C" long dlb_relbias_bwd_blocks(const RbArgs* a, int size);
extern "C" void dlb_relbias_bwd(const void* dout, int type, float* part,
                                void* dtable, int table_type, const RbArgs* a,
                                hipStream_t stream);

using torch::Tensor;
typedef c10::optional<Tensor> MaybeTensor;

static hipStream_t current_stream() {
  return at::hip::getCurrentHIPStream().stream();
}

static void launched() {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "kernel launch: ", hipGetErrorString(e));
}

// Rows are addressed from a tile's first one in 32 bits, 64 at a time.
static const int64_t PA_MAXSTRIDE = 1 << 24;

static PaTensor pa_tensor(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3 &&
                  t.scalar_type() == torch::kBFloat16,
              name, ": a bf16 GPU tensor [rows, heads, size] is wanted");
  TORCH_CHECK(t.size(2) == 1 || t.stride(2) == 1, name,
              ": the last dimension has to be dense");
  // the stride of a single row or head says nothing
  const int64_t row = t.size(0) > 1 ? t.stride(0) : 0;
  const int64_t head = t.size(1) > 1 ? t.stride(1) : 0;
  TORCH_CHECK(row >= 0 && row < PA_MAXSTRIDE && head >= 0, name,
              ": row stride out of range");
  return {t.data_ptr(), row, head};
}

// Bytes a load may have: the head size, the strides and the address are
// multiples of them.
static int pa_width(std::initializer_list<PaTensor> tensors, int64_t D) {
  int64_t all = D * 2;
  for (const auto& t : tensors)
    all |= (t.row | t.head) * 2 | (int64_t)reinterpret_cast<uintptr_t>(t.p);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

static void pa_bias(PaBias* b, const Tensor& table, int64_t H,
                    const std::vector<int64_t>& starts) {
  TORCH_CHECK(table.is_cuda() && table.is_contiguous() && table.dim() == 2 &&
                  table.size(1) == H &&
                  (size_t)table.size(0) == starts.size() &&
                  starts.size() >= 2 && starts.size() <= PA_MAXBUCKETS,
              "bias table: [buckets, heads], 2 to 256 buckets");
  TORCH_CHECK(table.scalar_type() == torch::kFloat32 ||
                  table.scalar_type() == torch::kBFloat16,
              "bias table: fp32 or bf16");
  b->table = table.data_ptr();
  b->buckets = (int)starts.size();
  b->is_bf16 = table.scalar_type() == torch::kBFloat16;
  for (size_t i = 0; i < starts.size(); ++i) b->starts[i] = (int)starts[i];
}

static void pa_check(const Tensor& q, const Tensor& k, const Tensor& v,
                     int64_t total) {
  TORCH_CHECK(k.sizes() == v.sizes() && q.size(0) == k.size(0) &&
                  q.size(2) == k.size(2) && k.size(1) >= 1 &&
                  q.size(1) % k.size(1) == 0 && q.size(2) >= 1 &&
                  q.size(2) <= 128 && total <= q.size(0) &&
                  q.size(0) < (1l << 31) / 2 && k.device() == q.device() &&
                  v.device() == q.device(),
              "packed attention: tensors do not fit");
}

// A work list: rows of 8, the chunks, then the joins; `slots` places for
// the sums of the chunks that are joined, `size` floats for each head's.
static PaWork pa_work(const Tensor& list, int64_t chunks, int64_t slots,
                      int64_t heads, int64_t size, const Tensor& like,
                      std::vector<Tensor>* keep) {
  TORCH_CHECK(list.device() == like.device() && list.is_contiguous() &&
                  list.scalar_type() == torch::kInt32 && list.dim() == 2 &&
                  list.size(1) == 8 && chunks >= 0 &&
                  chunks <= list.size(0) && slots >= 0 &&
                  list.size(0) * heads < (1l << 25) &&
                  chunks * heads < (1l << 24),  // workgroups of 256
              "packed attention: work list does not fit");
  // the list was made on another stream, maybe: it is not to be used again
  // before this one is done with it
  c10::hip::HIPCachingAllocator::recordStream(list.storage().data_ptr(),
                                              at::hip::getCurrentHIPStream());
  PaWork w{};
  w.chunks = static_cast<const PaChunk*>(list.data_ptr());
  w.joins = reinterpret_cast<const PaJoin*>(w.chunks + chunks);
  w.n_chunks = (int)chunks;
  w.n_joins = (int)(list.size(0) - chunks);
  if (slots > 0) {
    auto sums = torch::empty({slots * heads * (size + 256)},
                             like.options().dtype(torch::kFloat32));
    w.sums = sums.data_ptr<float>();
    w.rows = w.sums + slots * heads * size;
    keep->push_back(sums);
  }
  return w;
}

// Floats of a workgroup's accumulators, 128 rows of the padded head size.
static int64_t pa_tile(int64_t D) { return 128 * (D <= 64 ? 64 : 128); }

typedef std::tuple<Tensor, int64_t, int64_t> WorkList;  // chunks, slots
typedef c10::optional<WorkList> MaybeWork;

// q [T, H, D], k and v [T, Hkv, D]; work: the packing's query tiles.  Rows
// from `total` on belong to no sequence and come back as zeros.
static std::vector<Tensor> packed_attn_fwd(Tensor q, Tensor k, Tensor v,
                                           WorkList work, int64_t total,
                                           double scale, MaybeTensor table,
                                           std::vector<int64_t> starts) {
  pa_check(q, k, v, total);
  c10::DeviceGuard guard(q.device());
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  std::vector<Tensor> keep;
  PaFwd p{pa_tensor(q, "q"), pa_tensor(k, "k"), pa_tensor(v, "v")};
  auto o = torch::empty({T, H, D}, q.options());
  auto stats = torch::empty({H, T, table.has_value() ? 2 : 1},
                            q.options().dtype(torch::kFloat32));
  p.o = o.data_ptr();
  p.stats = stats.data_ptr<float>();
  p.work = pa_work(std::get<0>(work), std::get<1>(work), std::get<2>(work), H,
                   pa_tile(D), q, &keep);
  p.H = (int)H;
  p.G = (int)(H / k.size(1));
  p.D = (int)D;
  p.T = T;
  p.scale = (float)scale;
  PaBias bias{};
  if (table.has_value()) pa_bias(&bias, *table, H, starts);
  if (total < T) o.slice(0, total).zero_();
  if (p.work.n_chunks > 0) {
    dlb_packed_attn_fwd(&p, table.has_value() ? &bias : nullptr,
                        pa_width({p.q, p.k, p.v}, D), current_stream());
    launched();
  }
  return {o, stats};
}

// work_kv: the key tiles in steps of 64 queries for heads of up to 64, of
// 32 for others.  -> dq, dk, dv and, with a table and `table_grad`, its gradient.
static std::vector<Tensor> packed_attn_bwd(
    Tensor q, Tensor k, Tensor v, Tensor o, Tensor stats, Tensor go,
    WorkList work_q, WorkList work_kv, int64_t total, double scale,
    MaybeTensor table, std::vector<int64_t> starts, bool table_grad) {
  pa_check(q, k, v, total);
  c10::DeviceGuard guard(q.device());
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  TORCH_CHECK(go.sizes() == q.sizes() && go.device() == q.device() &&
              o.sizes() == q.sizes() && o.is_contiguous() &&
              stats.is_contiguous() &&
              stats.numel() == H * T * (table.has_value() ? 2 : 1));
  std::vector<Tensor> keep;
  PaBwd p{pa_tensor(q, "q"), pa_tensor(k, "k"), pa_tensor(v, "v"),
          pa_tensor(go, "gradient")};
  auto dq = torch::empty({T, H, D}, q.options());
  auto f32 = q.options().dtype(torch::kFloat32);
  auto delta = torch::empty({H, T}, f32);
  p.o = o.data_ptr();
  p.stats = stats.data_ptr<float>();
  p.delta = delta.data_ptr<float>();
  p.dq = dq.data_ptr();
  p.work_q = pa_work(std::get<0>(work_q), std::get<1>(work_q),
                     std::get<2>(work_q), H, pa_tile(D), q, &keep);
  p.H = (int)H;
  p.G = (int)(H / k.size(1));
  p.D = (int)D;
  p.T = T;
  p.scale = (float)scale;
  PaBias bias{};
  if (table.has_value()) pa_bias(&bias, *table, H, starts);
  const PaBias* b = table.has_value() ? &bias : nullptr;
  const int width = pa_width({p.q, p.k, p.v, p.go}, D);
  if (p.work_q.n_chunks > 0) {
    dlb_packed_attn_bwd_q(&p, b, width, current_stream());
    launched();
  }
  // the rest while that runs
  auto dk = torch::empty({T, k.size(1), D}, q.options());
  auto dv = torch::empty_like(dk);
  p.dk = dk.data_ptr();
  p.dv = dv.data_ptr();
  p.work_kv = pa_work(std::get<0>(work_kv), std::get<1>(work_kv),
                      std::get<2>(work_kv), k.size(1), 2 * pa_tile(D), q,
                      &keep);
  std::vector<Tensor> out = {dq, dk, dv};
  Tensor part, dtable;
  if (table.has_value() && table_grad) {
    part = torch::empty({p.work_kv.n_chunks, H, table->size(0)}, f32);
    dtable = torch::empty_like(*table);
    p.part = part.data_ptr<float>();
    out.push_back(dtable);
  }
  if (p.work_kv.n_chunks > 0) {
    dlb_packed_attn_bwd_kv(&p, b, width,
                           dtable.defined() ? dtable.data_ptr() : nullptr,
                           bias.is_bf16, current_stream());
    launched();
  } else if (dtable.defined()) {
    dtable.zero_();
  }
  if (total < T) {
    dq.slice(0, total).zero_();
    dk.slice(0, total).zero_();
    dv.slice(0, total).zero_();
  }
  return out;
}

static RbArgs rb_args(int64_t H, int64_t Q, int64_t K, int64_t buckets,
                      const std::vector<int64_t>& starts) {
  TORCH_CHECK(buckets >= 2 && buckets <= RB_MAXBUCKETS &&
                  ((int64_t)starts.size() == buckets ||
                   (int64_t)starts.size() * 2 == buckets),
              "position bias: 2 to 256 buckets");
  // 64 rows at least a workgroup where there are many
  TORCH_CHECK(H <= 65535 && Q <= 65535 * 64 && K < (1l << 31),
              "position bias: sizes out of range");
  RbArgs a;
  a.H = H;
  a.Q = Q;
  a.K = K;
  a.buckets = (int)buckets;
  a.side = (int)starts.size();
  a.both = a.side != a.buckets;
  for (size_t i = 0; i < starts.size(); ++i) a.starts[i] = (int)starts[i];
  return a;
}

static int rb_type(const Tensor& t) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == torch::kBFloat16 || s == torch::kFloat16 ||
                  s == torch::kFloat32,
              "position bias: bf16, fp16 or fp32");
  return s == torch::kBFloat16 ? 0 : s == torch::kFloat16 ? 1 : 2;
}

// table [buckets, H] -> [H, Q, K]; starts: least distance of each bucket of
// one side (half of the buckets if the sides are told apart).
static Tensor relbias_fwd(Tensor table, int64_t Q, int64_t K,
                          std::vector<int64_t> starts) {
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.is_contiguous());
  rb_type(table);
  c10::DeviceGuard guard(table.device());
  const RbArgs a = rb_args(table.size(1), Q, K, table.size(0), starts);
  auto out = torch::empty({a.H, Q, K}, table.options());
  if (out.numel() > 0) {
    dlb_relbias_fwd(table.data_ptr(), out.data_ptr(), &a,
                    (int)table.element_size(), current_stream());
    launched();
  }
  return out;
}

// dout [H, Q, K] -> [buckets, H] in the type of `table`.
static Tensor relbias_bwd(Tensor dout, Tensor table,
                          std::vector<int64_t> starts) {
  TORCH_CHECK(dout.is_cuda() && dout.dim() == 3 && dout.is_contiguous() &&
              dout.device() == table.device() && table.dim() == 2 &&
              table.size(1) == dout.size(0));
  c10::DeviceGuard guard(dout.device());
  // the kernel wants 16 bytes in a row: keys in front of the first, whose
  // gradient is 0, move no distance
  if (dout.size(2) > 0 && dout.size(2) < 8)
    dout = torch::constant_pad_nd(dout, {8 - dout.size(2), 0});
  const RbArgs a = rb_args(dout.size(0), dout.size(1), dout.size(2),
                           table.size(0), starts);
  auto dtable = torch::empty({table.size(0), a.H}, table.options());
  if (dout.numel() == 0) return dtable.zero_();
  auto part = torch::empty(
      {dlb_relbias_bwd_blocks(&a, (int)dout.element_size()), a.H,
       table.size(0)},
      dout.options().dtype(torch::kFloat32));
  dlb_relbias_bwd(dout.data_ptr(), rb_type(dout), part.data_ptr<float>(),
                  dtable.data_ptr(), rb_type(table), &a, current_stream());
  launched();
  return dtable;
}

// ---- autograd.  In C++, where a call and its gradient cost the host a
// third of what Python functions do: small sequences are bound by it.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients under create_graph: differentiating them again is an error.
static variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " can be differentiated once only",
      (int64_t)grads.size());
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  return (*error)(std::move(grads));
}

// A backward under capture hands its gradients to the nodes of its inputs.
// One that an eager graph made on the default stream (the accumulator of a
// leaf lives as long as a graph that reads the leaf) would draw that stream
// into the capture, which ends the process: an error here instead.
static void refuse_eager_inputs(const char* name) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() ==
      c10::hip::CaptureStatus::None)
    return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    if (!node->task_should_compute_output(i)) continue;
    const auto stream = node->next_edge(i).function->stream();
    TORCH_CHECK(!stream.has_value() || stream->id() != 0, name,
                ": a backward pass is captured while an eager graph of the "
                "same tensors is alive; drop that graph's results first");
  }
}

// A tensor the kernels can read: itself, if its strides allow it.
static Tensor readable(const Tensor& t) {
  return (t.size(2) == 1 || t.stride(2) == 1) &&
                 (t.size(0) <= 1 || t.stride(0) < PA_MAXSTRIDE)
             ? t
             : t.contiguous();
}

struct PackedAttention
    : public torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0,
                        const Tensor& k0, const Tensor& v0,
                        const MaybeTensor& table0, WorkList work_q,
                        MaybeWork work_kv, int64_t total, double scale,
                        std::vector<int64_t> starts, bool table_grad) {
    const Tensor q = readable(q0), k = readable(k0), v = readable(v0);
    MaybeTensor table;
    if (table0.has_value()) table = table0->contiguous();
    auto out = packed_attn_fwd(q, k, v, work_q, total, scale, table, starts);
    ctx->save_for_backward({q, k, v, out[0], out[1],
                            table.has_value() ? *table : Tensor(),
                            std::get<0>(work_q),
                            work_kv ? std::get<0>(*work_kv) : Tensor()});
    auto& d = ctx->saved_data;
    d["counts"] = std::vector<int64_t>{
        std::get<1>(work_q), std::get<2>(work_q),
        work_kv ? std::get<1>(*work_kv) : 0,
        work_kv ? std::get<2>(*work_kv) : 0, total};
    d["scale"] = scale;
    d["starts"] = std::move(starts);
    d["table_grad"] = table_grad;
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    refuse_eager_inputs("packed_causal_attention");
    const auto saved = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    const auto n = d["counts"].toIntVector();
    const bool table_grad = d["table_grad"].toBool();
    MaybeTensor table;
    if (saved[5].defined()) table = saved[5];
    variable_list out(10);
    {
      at::AutoGradMode off(false);
      auto grads = packed_attn_bwd(
          saved[0], saved[1], saved[2], saved[3], saved[4],
          readable(grad[0]), WorkList{saved[6], n[0], n[1]},
          WorkList{saved[7], n[2], n[3]}, n[4], d["scale"].toDouble(), table,
          d["starts"].toIntVector(), table_grad);
      for (size_t i = 0; i < grads.size(); ++i) out[i] = grads[i];
    }
    return once(std::move(out), "packed_causal_attention");
  }
};

static Tensor packed_attention(Tensor q, Tensor k, Tensor v,
                               MaybeTensor table, WorkList work_q,
                               MaybeWork work_kv, int64_t total, double scale,
                               std::vector<int64_t> starts) {
  return PackedAttention::apply(
      q, k, v, table, work_q, work_kv, total, scale, starts,
      table.has_value() && table->requires_grad());
}

struct PositionBias : public torch::autograd::Function<PositionBias> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, int64_t Q,
                        int64_t K, std::vector<int64_t> starts,
                        at::ScalarType type) {
    ctx->save_for_backward({table});
    auto out = relbias_fwd(table.to(type).contiguous(), Q, K, starts);
    ctx->saved_data["starts"] = std::move(starts);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    refuse_eager_inputs("relative_position_bias");
    variable_list out(5);
    {
      at::AutoGradMode off(false);
      out[0] = relbias_bwd(grad[0].contiguous(),
                           ctx->get_saved_variables()[0],
                           ctx->saved_data["starts"].toIntVector());
    }
    return once(std::move(out), "relative_position_bias");
  }
};

static Tensor position_bias(Tensor table, int64_t Q, int64_t K,
                            std::vector<int64_t> starts,
                            py::object type) {
  return PositionBias::apply(table, Q, K, starts,
                             torch::python::detail::py_object_to_dtype(type));
}

void bind_longctx(py::module_& m) {
  m.def("packed_attention", &packed_attention,
        "causal attention over packed sequences, differentiable");
  m.def("position_bias", &position_bias,
        "bucketed position bias as a grid, differentiable in its table");
  m.def("packed_attn_fwd", &packed_attn_fwd,
        "causal attention over packed sequences");
  m.def("packed_attn_bwd", &packed_attn_bwd,
        "its gradients, from the saved row statistics");
  m.def("relbias_fwd", &relbias_fwd, "bucketed position bias, [H, Q, K]");
  m.def("relbias_bwd", &relbias_bwd, "gradient of its table");
}
