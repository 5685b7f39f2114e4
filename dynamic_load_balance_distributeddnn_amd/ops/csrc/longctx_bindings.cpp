// Python bindings of packed causal attention and of the position bias.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include "longctx_args.h"

extern "C" void dlb_packed_attn_fwd(const PaFwd* p, const PaBias* bias,
                                    long items, int vec, hipStream_t stream);
extern "C" void dlb_packed_attn_bwd(const PaBwd* p, const PaBias* bias,
                                    const PaItem* items_kv, long items,
                                    int vec, void* dtable, int dtable_bf16,
                                    hipStream_t stream);
extern "C" void dlb_relbias_fwd(const void* table, void* out, const RbArgs* a,
                                int size, hipStream_t stream);
extern "C" long dlb_relbias_bwd_blocks(const RbArgs* a);
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

static PaTensor pa_tensor(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3 &&
                  t.scalar_type() == torch::kBFloat16,
              name, ": a bf16 GPU tensor [rows, heads, size] is wanted");
  TORCH_CHECK(t.size(2) == 1 || t.stride(2) == 1, name,
              ": the last dimension has to be dense");
  // 64 rows are addressed from one base in 32 bits
  TORCH_CHECK(t.stride(0) >= 0 && t.stride(0) < (1 << 24) && t.stride(1) >= 0,
              name, ": row stride out of range");
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

// 16-byte loads: the head size, the strides and the address allow them.
static bool pa_vec(const PaTensor& t, int64_t D) {
  return D % 8 == 0 && t.row % 8 == 0 && t.head % 8 == 0 &&
         reinterpret_cast<uintptr_t>(t.p) % 16 == 0;
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
                     const Tensor& items, int64_t total) {
  TORCH_CHECK(k.sizes() == v.sizes() && q.size(0) == k.size(0) &&
                  q.size(2) == k.size(2) && k.size(1) >= 1 &&
                  q.size(1) % k.size(1) == 0 && q.size(2) >= 1 &&
                  q.size(2) <= 128 && total <= q.size(0) &&
                  q.size(0) < (1l << 31) / 2,
              "packed attention: shapes do not fit");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device() &&
                  items.device() == q.device() && items.is_contiguous() &&
                  items.scalar_type() == torch::kInt32 && items.dim() == 2 &&
                  items.size(1) == 4 &&
                  items.size(0) * q.size(1) < (1l << 31),
              "packed attention: work items do not fit");
}

// q [T, H, D], k and v [T, Hkv, D]; items: the packing's row tiles.  Rows
// from `total` on belong to no sequence and come back as zeros.
static std::vector<Tensor> packed_attn_fwd(Tensor q, Tensor k, Tensor v,
                                           Tensor items, int64_t total,
                                           double scale, MaybeTensor table,
                                           std::vector<int64_t> starts) {
  pa_check(q, k, v, items, total);
  c10::DeviceGuard guard(q.device());
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  PaFwd p{pa_tensor(q, "q"), pa_tensor(k, "k"), pa_tensor(v, "v")};
  auto o = torch::empty({T, H, D}, q.options());
  auto stats = torch::empty({H, T, table.has_value() ? 2 : 1},
                            q.options().dtype(torch::kFloat32));
  p.o = o.data_ptr();
  p.stats = stats.data_ptr<float>();
  p.items = static_cast<const PaItem*>(items.data_ptr());
  p.H = (int)H;
  p.G = (int)(H / k.size(1));
  p.D = (int)D;
  p.T = T;
  p.scale = (float)scale;
  PaBias bias{};
  if (table.has_value()) pa_bias(&bias, *table, H, starts);
  if (total < T) o.slice(0, total).zero_();
  if (items.size(0) * H > 0) {
    const bool vec = pa_vec(p.q, D) && pa_vec(p.k, D) && pa_vec(p.v, D);
    dlb_packed_attn_fwd(&p, table.has_value() ? &bias : nullptr,
                        items.size(0), vec, current_stream());
    launched();
  }
  return {o, stats};
}

// -> dq, dk, dv and, with a table and `table_grad`, its gradient.
static std::vector<Tensor> packed_attn_bwd(
    Tensor q, Tensor k, Tensor v, Tensor o, Tensor stats, Tensor go,
    Tensor items, Tensor items_kv, int64_t total, double scale,
    MaybeTensor table, std::vector<int64_t> starts, bool table_grad) {
  pa_check(q, k, v, items, total);
  pa_check(q, k, v, items_kv, total);
  c10::DeviceGuard guard(q.device());
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  TORCH_CHECK(go.sizes() == q.sizes() && o.sizes() == q.sizes() &&
              o.is_contiguous() && stats.is_contiguous() &&
              stats.numel() == H * T * (table.has_value() ? 2 : 1) &&
              items.size(0) == items_kv.size(0));
  PaBwd p{pa_tensor(q, "q"), pa_tensor(k, "k"), pa_tensor(v, "v"),
          pa_tensor(go, "gradient")};
  auto dq = torch::empty({T, H, D}, q.options());
  auto dk = torch::empty({T, k.size(1), D}, q.options());
  auto dv = torch::empty_like(dk);
  auto f32 = q.options().dtype(torch::kFloat32);
  auto delta = torch::empty({H, T}, f32);
  p.o = o.data_ptr();
  p.stats = stats.data_ptr<float>();
  p.delta = delta.data_ptr<float>();
  p.dq = dq.data_ptr();
  p.dk = dk.data_ptr();
  p.dv = dv.data_ptr();
  p.items = static_cast<const PaItem*>(items.data_ptr());
  p.H = (int)H;
  p.G = (int)(H / k.size(1));
  p.D = (int)D;
  p.T = T;
  p.scale = (float)scale;
  std::vector<Tensor> out = {dq, dk, dv};
  PaBias bias{};
  Tensor part, dtable;
  if (table.has_value()) {
    pa_bias(&bias, *table, H, starts);
    if (table_grad) {
      part = torch::empty({items.size(0), H, table->size(0)}, f32);
      dtable = torch::empty_like(*table);
      p.part = part.data_ptr<float>();
      out.push_back(dtable);
    }
  }
  if (total < T) {
    dq.slice(0, total).zero_();
    dk.slice(0, total).zero_();
    dv.slice(0, total).zero_();
  }
  if (items.size(0) * H > 0) {
    const bool vec = pa_vec(p.q, D) && pa_vec(p.k, D) && pa_vec(p.v, D) &&
                     pa_vec(p.go, D);
    dlb_packed_attn_bwd(&p, table.has_value() ? &bias : nullptr,
                        static_cast<const PaItem*>(items_kv.data_ptr()),
                        items.size(0), vec,
                        table_grad ? dtable.data_ptr() : nullptr,
                        bias.is_bf16, current_stream());
    launched();
  } else if (table_grad) {
    dtable.zero_();
  }
  return out;
}

static RbArgs rb_args(int64_t H, int64_t Q, int64_t K, int64_t buckets,
                      const std::vector<int64_t>& starts) {
  TORCH_CHECK(buckets >= 2 && buckets <= RB_MAXBUCKETS &&
                  ((int64_t)starts.size() == buckets ||
                   (int64_t)starts.size() * 2 == buckets),
              "position bias: 2 to 256 buckets");
  TORCH_CHECK(H <= 65535 && Q < (1 << 22) && K < (1l << 31),
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
  const RbArgs a = rb_args(dout.size(0), dout.size(1), dout.size(2),
                           table.size(0), starts);
  auto dtable = torch::empty({table.size(0), a.H}, table.options());
  if (dout.numel() == 0) return dtable.zero_();
  auto part = torch::empty({dlb_relbias_bwd_blocks(&a), a.H, table.size(0)},
                           dout.options().dtype(torch::kFloat32));
  dlb_relbias_bwd(dout.data_ptr(), rb_type(dout), part.data_ptr<float>(),
                  dtable.data_ptr(), rb_type(table), &a, current_stream());
  launched();
  return dtable;
}

void bind_longctx(py::module_& m) {
  m.def("packed_attn_fwd", &packed_attn_fwd,
        "causal attention over packed sequences");
  m.def("packed_attn_bwd", &packed_attn_bwd,
        "its gradients, from the saved row statistics");
  m.def("relbias_fwd", &relbias_fwd, "bucketed position bias, [H, Q, K]");
  m.def("relbias_bwd", &relbias_bwd, "gradient of its table");
}
