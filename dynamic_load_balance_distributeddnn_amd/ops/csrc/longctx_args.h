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

// Work item: one row tile of one sequence.
struct PaItem {
  int first;  // the sequence's first row
  int len;    // and its rows
  int tile;   // which tile of 128 rows
  int pad;
};

struct PaFwd {
  PaTensor q, k, v;
  void* o;        // [T, H, D]
  float* stats;   // [H, T]: log2 of the row's sum of exponentials;
                  // with bias [H, T, 2]: maximum, log2 of the sum
  const PaItem* items;
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
  float* part;         // [items, H, buckets] of the table's gradient
  const PaItem* items;
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
