// kvcache.hpp -- a paged key-value cache and the operators of a decode step over it.
//
// No counterpart in the reference, whose MHA layer rebuilds its ring of keys and values inside
// every forward (src/layers/mha/mha.cpp:123-183). The pages, the page table and the lengths are
// the caller's device memory; the handle holds their description, the launches' workspaces and
// an error word. Calls on one handle must not overlap each other.
#pragma once

#include "common.hpp"

#include <vector>

namespace wb {

// Storage types of the pages (ids of the reference's DType table).
enum class KvType : int32_t { F32 = 1, F16 = 2, BF16 = 3, E4M3 = 4 };

inline int kv_size(KvType t) { return t == KvType::F32 ? 4 : (t == KvType::E4M3 ? 1 : 2); }

// One pool: element (page p, slot s, head h, dim d) lies at base[p * page + s * slot + h * head + d]
// (strides in elements).
struct KvPool {
  uint8_t* base = nullptr;
  int64_t page = 0, slot = 0, head = 0;
};

// What every kernel gets. max_slots = pages_per_seq * page_size; the per-slot records weights and
// positions are [num_seqs][num_kv][max_slots].
struct KvView {
  KvPool k, v;
  float k_scale = 1.0f, v_scale = 1.0f;  // value = stored * scale
  int num_heads = 0, num_kv = 0, head_dim = 0, page_size = 0, num_pages = 0, num_seqs = 0, pages_per_seq = 0;
  int64_t table_stride = 0;
  const int32_t* table = nullptr;
  int32_t* lens = nullptr;       // slots in use
  int32_t* seen = nullptr;       // tokens seen (= lens when the caller keeps none)
  float* weights = nullptr;      // accumulated attention weight of a slot (may be null)
  int32_t* positions = nullptr;  // token position held by a slot (null: the slot index)
  int max_slots = 0;
  int* err = nullptr;
};

// Error codes that kernels leave in the error word.
constexpr int kKvErrPage = 1;  // a page id of the table outside [0, num_pages)
constexpr int kKvErrSlot = 2;  // a length outside [0, max_slots], or an append past the last slot
constexpr int kKvErrHeld = 3;  // a prompt for a sequence that holds slots already
constexpr int kKvErrRows = 4;  // cu decreases, is negative or goes past the rows

struct KvCache {
  int device = 0;
  KvType type = KvType::BF16;
  KvView view;
  double theta = 0.0;            // rotary base that inv_turns was made for
  std::vector<double> inv_turns;  // half turns (units of pi) per position of each rotary pair
  uint8_t* work = nullptr;       // the one allocation behind what follows
  int* err = nullptr;
  int* ticket = nullptr;         // block counter of append (zero between calls)
  int32_t* step_lens = nullptr;  // [num_seqs] lengths of a step that leaves sequences out
  // attend (kv_attend.cu)
  bool attend_tiled = false;
  int attend_blocks = 0;         // blocks of the tiled form
  int attend_cluster = 0;        // blocks of a unit's cluster (0: runs of tiles)
  size_t part_bytes = 0, span_bytes = 0;
  float* part = nullptr;         // partial results
  void* spans = nullptr;         // where each unit's parts are
  float* scores = nullptr;       // [num_seqs][num_heads][max_slots]; with weights only
  float* lse = nullptr;          // [num_seqs][num_heads]
  int32_t* moves = nullptr;      // evict: [num_seqs][num_kv][2][max_slots / 2] slots to fill, slots to take
  int32_t* n_moves = nullptr;    // [num_seqs][num_kv]
  int* evict_tickets = nullptr;  // [num_seqs], zero between calls
  ~KvCache();
};

Status kv_create(int device, KvType type, const KvView& view, KvCache** out);

// Picks the form of attend and sizes its workspaces (kv_create).
Status attend_plan(KvCache* c);

struct KvAppendArgs {
  int rows = 0;
  const float* k = nullptr;
  const float* v = nullptr;
  const float* q = nullptr;  // may be null
  float* q_out = nullptr;
  int64_t k_ld = 0, v_ld = 0, q_ld = 0, q_out_ld = 0;
  const int32_t* cu = nullptr;  // [num_seqs + 1] first row of each sequence; null: one row each
  int only = -1;                // >= 0: every row is this sequence's, a prompt from position 0 (cu, start,
                                // start_seen null); one that holds slots already is left as it is
  double theta = 0.0;           // <= 0: no rotation
  const int32_t* start = nullptr;       // slots in use before the call (null: lens)
  const int32_t* start_seen = nullptr;  // tokens seen before the call (null: seen)
  const int32_t* active = nullptr;      // [num_seqs]; 0: this sequence's row is left out (cu null, only < 0)
  int32_t* step_lens = nullptr;         // with active: lens, 0 for a sequence that is left out
};
Status kv_append(KvCache* c, const KvAppendArgs& a, cudaStream_t st);

struct KvAttendArgs {
  const float* q = nullptr;  // [num_seqs][num_heads][head_dim], rows q_ld apart
  float* out = nullptr;
  int64_t q_ld = 0, out_ld = 0;
  float scale = 0.0f;  // <= 0: 1 / sqrt(head_dim)
  int window = 0;      // > 0: only positions > query position - window
  int alibi = 0;
  int accumulate = 0;  // weights = weights_in + this step's attention weights
  const float* weights_in = nullptr;  // null: weights
  const int32_t* lens = nullptr;      // slots to attend to (null: the cache's lens)
};
Status kv_attend(KvCache* c, const KvAttendArgs& a, cudaStream_t st);

struct KvEvictArgs {
  int keep = 0, budget = 0, sinks = 0, recent = 0;
  const int32_t* lens_in = nullptr;  // null: lens / weights / positions themselves
  const float* weights_in = nullptr;
  const int32_t* positions_in = nullptr;
};
Status kv_evict(KvCache* c, const KvEvictArgs& a, cudaStream_t st);

// Synchronizes the stream; reports and clears the error word.
Status kv_check_error(KvCache* c, cudaStream_t st);

inline bool pool_aligned(const KvPool& p, int size, int bytes) {
  return reinterpret_cast<uintptr_t>(p.base) % bytes == 0 && p.page * size % bytes == 0 && p.slot * size % bytes == 0 &&
         p.head * size % bytes == 0;
}

} // namespace wb
