// Arguments of the packed attention and position bias launchers, shared by
// the kernels and the host binding (no device types).
#pragma once

#define PA_MAXBUCKETS 256
#define RB_MAXBUCKETS 256

// One [rows, heads, D] bf16 tensor: element strides, the last one 1.
struct PaTensor {
  const void* p;
  long row;
  long head;
};

// The bias table of a launch: [buckets, heads], fp32 or bf16.
struct PaBias {
  const void* table;
  int buckets;
  int is_bf16;
  int starts[PA_MAXBUCKETS];  // least distance of each bucket
};

// Part of one 128-row tile's work: of a query tile the key tiles (64 keys)
// begin .. end - 1, of a key tile that many steps (32 queries of a head).
struct PaChunk {
  int first;  // the sequence's first row
  int len;    // and its rows
  int tile;
  int begin, end;
  int slot;   // where its sums go, -1: they are the whole tile's
  int pad[2];
};

// A tile in several chunks: their slots are slot .. slot + n - 1.
struct PaJoin {
  int first, len, tile;
  int slot, n;
  int pad[3];
};

struct PaWork {
  const PaChunk* chunks;  // most work first
  const PaJoin* joins;
  int n_chunks, n_joins;
  float* sums;   // [slots, heads] of a workgroup's accumulators
  float* rows;   // [slots, heads, 128, 2] of its row statistics
};

struct PaFwd {
  PaTensor q, k, v;
  void* o;        // [T, H, D]
  float* stats;   // [H, T]: log2 of the row's sum of exponentials;
                  // with bias [H, T, 2]: maximum, log2 of the sum
  PaWork work;
  int H, G, D;    // heads, heads per key/value head, head size
  long T;
  float scale;
};

struct PaBwd {
  PaTensor q, k, v, go;
  const void* o;       // [T, H, D]
  const float* stats;  // as the forward left them
  float* delta;        // [H, T]
  void *dq, *dk, *dv;  // [T, H, D], [T, H / G, D] twice
  float* part;         // [key chunks, H, buckets] of the table's gradient
  PaWork work_q, work_kv;
  int H, G, D;
  long T;
  float scale;
};

struct RbArgs {
  long H, Q, K;
  int buckets;  // of the table
  int side;     // of one direction: half of them if both are told apart
  int both;
  int starts[RB_MAXBUCKETS];  // least distance of each bucket of a side
};
