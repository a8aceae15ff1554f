// ops.h -- the argument blocks and entry points of the serving operators (tilelang._tl_ops).
//
// Every operator has one argument block, filled and checked by bindings.cpp from torch tensors, and two
// entry points that read it: *_hip launches hand-written gfx950 kernels on a stream, *_cpu computes the same
// definition on the host.  Pointers are device pointers for the first and host pointers for the second.
// Strides count elements.
#pragma once

#include <cstdint>

struct ihipStream_t;

namespace tl_ops {

using Stream = ihipStream_t*;

enum Type : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// --------------------------------------------------------------------------------------- norm

// h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, q = e4m3(y / scale) with one scale per `group`
struct NormQuantArgs {
  const void* x;
  const void* residual;  // or null
  const void* weight;
  int64_t x_stride, residual_stride;
  uint8_t* q;    // [rows, width]
  float* scale;  // [rows, width / group]
  void* h;       // [rows, width], or null: not wanted
  void* y;       // [rows, width], or null: not wanted
  int64_t rows;
  int width, group;
  float eps;
  bool pow2;
  Type type;
};

constexpr int kNormMaxWidth = 65536;

void norm_quant_hip(const NormQuantArgs&, Stream);
void norm_quant_cpu(const NormQuantArgs&);

// --------------------------------------------------------------------------------------- cache

// The pools: K [pages, heads, page, wide], V [pages, heads, wide, page], scales [pages, heads].
struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  const int* table;  // [batch, table_width], rows table_stride apart
  const int* lengths;
  int64_t pages, table_stride;
  int table_width, heads, dim, wide, page_shift;
};

struct AppendArgs {
  Cache cache;
  const void* x[2];  // K's and V's new tokens, [batch, new_tokens, heads, dim]
  int64_t stride_b[2], stride_t[2], stride_h[2];
  int batch, new_tokens;
  Type type;
};

void kv_append_hip(const AppendArgs&, Stream);
void kv_append_cpu(const AppendArgs&);

struct AttentionArgs {
  Cache cache;
  const void* q;  // [batch, new_tokens, heads, dim]
  int64_t stride_b, stride_t, stride_h;
  void* out;   // contiguous, as q
  float* lse;  // [batch, new_tokens, heads], or null
  int batch, new_tokens, heads;
  float scale;
  Type type;
  int tile, splits;  // rows of a workgroup and parts of the key axis: kv_attention_plan()
  float* part_o;   // splits > 1: [batch * new_tokens * heads, splits, dim]
  float* part_ml;  // splits > 1: [batch * new_tokens * heads, splits, 2]
};

void kv_attention_plan(AttentionArgs&, int64_t longest);  // longest: the tokens that a sequence has at most
void kv_attention_hip(const AttentionArgs&, Stream);
void kv_attention_cpu(const AttentionArgs&);

// --------------------------------------------------------------------------------------- beams

struct BeamArgs {
  const void* logits;  // [batch * beams, vocab], rows stride apart
  int64_t stride;
  const float* scores;      // [batch, beams]
  const uint8_t* finished;  // [batch, beams], or null
  int64_t eos;
  float* out_scores;     // [batch, take]
  int64_t* out_parents;  // [batch, take]
  int64_t* out_tokens;   // [batch, take]
  int64_t batch;
  int beams, take, vocab;
  Type type;
  int chunks;           // parts of the vocabulary: beam_select_chunks()
  float* part_stat;     // [batch * beams, chunks, waves, 2]
  uint64_t* part_list;  // [batch * beams, chunks, take]
};

constexpr int kBeamMaxTake = 64;
constexpr int kBeamMaxBeams = 64;
constexpr int kBeamMaxVocab = 1 << 20;
constexpr int kBeamMaxLists = 4096;  // beams * chunks

int beam_select_chunks(int vocab);
int64_t beam_select_scratch(int64_t rows, int chunks, int take);  // 8-byte words of scratch memory
void beam_select_hip(BeamArgs, uint64_t* scratch, Stream);
void beam_select_cpu(const BeamArgs&);

struct ReorderState {
  uint8_t* data;
  int64_t stride;  // bytes between two rows
  int64_t bytes;   // bytes of a row that move
  int64_t first;   // the first of its workgroups
};

constexpr int kReorderMaxBeams = 32;
constexpr int kReorderStates = 96;  // states that one launch takes
// and bytes of their rows: a wave moves 1024 of them, and a launch has fewer than 2^32 threads
constexpr int64_t kReorderMaxBytes = (int64_t(1) << 36) - 1024;

struct ReorderArgs {
  ReorderState state[kReorderStates];
  const int64_t* parents;  // [batch, beams]
  int64_t batch;
  int beams, states;
};

void reorder_hip(ReorderArgs, Stream);
void reorder_cpu(const ReorderArgs&);

}  // namespace tl_ops
