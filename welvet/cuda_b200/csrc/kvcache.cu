// kvcache.cu -- append and eviction over a paged key-value cache, and its handle (sm_100a).
#include "kvcache.hpp"
#include "kvcache.cuh"

#include <cmath>

namespace wb {
namespace {

// ---------------------------------------------------------------- append

// Rotary angles are position * theta^(-2i/D); the host passes them in half turns (angle / pi) so
// that the kernel reduces the product in 64 bits by one rint and calls sincospif on [-1, 1]: the
// angle is good to 2^-24 at any position, which 32 bits would lose past position 10^3.
constexpr int kMaxPairs = 128;
struct RopeTable {
  double turns[kMaxPairs];
};

struct AppendParams {
  KvAppendArgs a;
  KvView c;
  int half;  // rotary pairs (0: no rotation)
  int* ticket;
  RopeTable rope;
};

constexpr int kAppendThreads = 256;

// One block per new token: the token's angles once into shared memory, then its key, value and
// query heads, pair (d, d + half) by pair. HBM bound: 4 B read per element, the page's type
// written (and 4 B for q). kVec: four consecutive pairs a thread (16-byte accesses).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAppendThreads) k_append(const __grid_constant__ AppendParams p) {
  __shared__ float s_cos[kMaxPairs], s_sin[kMaxPairs];
  __shared__ int s_last;
  const KvView& c = p.c;
  const int t = blockIdx.x;
  const int D = c.head_dim, half = p.half;
  // the row's sequence: the last s with cu[s] <= t
  int seq = t, i = 0;
  bool live = t < p.a.rows;
  if (p.a.cu) {
    int lo = 0, hi = c.num_seqs;  // cu[lo] <= t < cu[hi] is what a row of a sequence has
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.a.cu[mid] <= t) lo = mid; else hi = mid;
    }
    seq = lo;
    i = t - p.a.cu[seq];
    live = live && i >= 0 && t < p.a.cu[seq + 1];
  }
  if (live) {
    const int64_t slot = static_cast<int64_t>(p.a.start[seq]) + i;
    const int64_t pos = static_cast<int64_t>(p.a.start_seen[seq]) + i;
    int64_t page = -1;
    if (slot >= 0 && slot < c.max_slots) {
      page = c.table[seq * c.table_stride + slot / c.page_size];
      if (page < 0 || page >= c.num_pages) {
        page = -1;
        if (threadIdx.x == 0) atomicCAS(c.err, 0, kKvErrPage);
      }
    } else if (threadIdx.x == 0) {
      atomicCAS(c.err, 0, kKvErrSlot);
    }
    for (int d = threadIdx.x; d < half; d += kAppendThreads) {
      const double u = static_cast<double>(pos) * p.rope.turns[d];
      sincospif(static_cast<float>(u - 2.0 * rint(0.5 * u)), &s_sin[d], &s_cos[d]);
    }
    __syncthreads();
    const int in_page = static_cast<int>(slot % c.page_size);
    T* kd = reinterpret_cast<T*>(c.k.base) + page * c.k.page + in_page * c.k.slot;
    T* vd = reinterpret_cast<T*>(c.v.base) + page * c.v.page + in_page * c.v.slot;
    const float ks = 1.0f / c.k_scale, vs = 1.0f / c.v_scale;
    const float* k = p.a.k + t * p.a.k_ld;
    const float* v = p.a.v + t * p.a.v_ld;
    const float* q = p.a.q ? p.a.q + t * p.a.q_ld : nullptr;
    float* qo = p.a.q_out + t * p.a.q_out_ld;
    const int heads = 2 * c.num_kv + (q ? c.num_heads : 0);
    if constexpr (kVec) {
      // a thread takes 4 dims of the lower half and their partners (values: 4 + 4 dims)
      const int per = D / 8, h2 = D / 2;
      for (int w = threadIdx.x; w < heads * per; w += kAppendThreads) {
        const int h = w / per, d = 4 * (w - h * per);
        const bool is_v = h >= c.num_kv && h < 2 * c.num_kv;
        const float* src = h < c.num_kv ? k + h * D : (is_v ? v + (h - c.num_kv) * D : q + (h - 2 * c.num_kv) * D);
        const float4 lo = *reinterpret_cast<const float4*>(src + d);
        const float4 hi = *reinterpret_cast<const float4*>(src + d + h2);
        float a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
        if (!is_v && half > 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float cs = s_cos[d + e], sn = s_sin[d + e], x0 = a[e], x1 = b[e];
            a[e] = x0 * cs - x1 * sn;
            b[e] = x0 * sn + x1 * cs;
          }
        }
        if (h >= 2 * c.num_kv) {
          float* o = qo + (h - 2 * c.num_kv) * D;
          *reinterpret_cast<float4*>(o + d) = make_float4(a[0], a[1], a[2], a[3]);
          *reinterpret_cast<float4*>(o + d + h2) = make_float4(b[0], b[1], b[2], b[3]);
        } else if (page >= 0) {
          T* o = is_v ? vd + (h - c.num_kv) * c.v.head : kd + h * c.k.head;
          const float s = is_v ? vs : ks;
          store4<T>(o + d, a, s);
          store4<T>(o + d + h2, b, s);
        }
      }
    } else {
      for (int w = threadIdx.x; w < heads * D; w += kAppendThreads) {
        const int h = w / D, d = w - h * D;
        const bool is_v = h >= c.num_kv && h < 2 * c.num_kv;
        const float* src = h < c.num_kv ? k + h * D : (is_v ? v + (h - c.num_kv) * D : q + (h - 2 * c.num_kv) * D);
        float x = src[d];
        if (!is_v && d < 2 * half) {
          const int e = d < half ? d : d - half;
          const float other = src[d < half ? d + half : e];
          x = d < half ? x * s_cos[e] - other * s_sin[e] : other * s_sin[e] + x * s_cos[e];
        }
        if (h >= 2 * c.num_kv) qo[(h - 2 * c.num_kv) * D + d] = x;
        else if (page >= 0) {
          if (is_v) vd[(h - c.num_kv) * c.v.head + d] = to_stored<T>(x * vs);
          else kd[h * c.k.head + d] = to_stored<T>(x * ks);
        }
      }
    }
    if (slot >= 0 && slot < c.max_slots) {
      for (int h = threadIdx.x; h < c.num_kv; h += kAppendThreads) {
        const int64_t at = (static_cast<int64_t>(seq) * c.num_kv + h) * c.max_slots + slot;
        if (c.positions) c.positions[at] = static_cast<int32_t>(pos);
        if (c.weights) c.weights[at] = 0.0f;
      }
    }
  }
  // The last block to finish advances the lengths: start may be lens itself, which every block
  // has read by then.
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (threadIdx.x == 0) *p.ticket = 0;
  for (int s = threadIdx.x; s < c.num_seqs; s += kAppendThreads) {
    const int n = p.a.cu ? p.a.cu[s + 1] - p.a.cu[s] : 1;
    const int64_t len = static_cast<int64_t>(p.a.start[s]) + n, tot = static_cast<int64_t>(p.a.start_seen[s]) + n;
    c.lens[s] = static_cast<int32_t>(len < c.max_slots ? len : c.max_slots);
    if (c.seen != c.lens) c.seen[s] = static_cast<int32_t>(tot);
  }
}

// ---------------------------------------------------------------- eviction

struct EvictParams {
  KvEvictArgs a;
  KvView c;
  int32_t* moves;
  int32_t* n_moves;
};

constexpr int kEvictThreads = 1024;
constexpr int kRadixBits = 11;  // three passes over a 32-bit key: 11 + 11 + 10 bits

// The order in which slots stay: protected ones first, then by weight; larger keys stay. NaN counts
// as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t evict_key(const EvictParams& p, int64_t rec, int j, int seen) {
  const int pos = p.a.positions_in[rec + j];
  if (pos < p.a.sinks || pos >= seen - p.a.recent) return 0xffffffffu;
  const float w = p.a.weights_in[rec + j];
  if (isnan(w)) return 0x007fffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive sum of v over the block's threads; *total the whole sum.
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[w] = x;
  __syncthreads();
  if (w == 0) {
    int y = lane < static_cast<int>(blockDim.x) / 32 ? s_warp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    s_warp[lane] = y;
  }
  __syncthreads();
  *total = s_warp[31];
  return x - v + (w > 0 ? s_warp[w - 1] : 0);
}

// One block per (sequence, kv head): the keep-th largest key by radix selection, then, in slot
// order, the slots below keep that go (to fill) and those above it that stay (to take). Both
// lists are equally long, and no slot is in both, so the moves can run in any order.
__global__ void __launch_bounds__(kEvictThreads) k_evict_select(const __grid_constant__ EvictParams p) {
  __shared__ int hist[1 << kRadixBits];
  __shared__ int s_warp[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_rest;
  const KvView& c = p.c;
  const int kv = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int row = b * c.num_kv + kv;
  const int64_t rec = static_cast<int64_t>(row) * c.max_slots;
  int len = p.a.lens_in[b];
  if (len < 0 || len > c.max_slots) {
    if (tid == 0) atomicCAS(c.err, 0, kKvErrSlot);
    len = len < 0 ? 0 : c.max_slots;
  }
  const bool cut = len > p.a.budget;
  const int keep = p.a.keep, seen = c.seen[b];
  if (p.a.weights_in != c.weights || p.a.positions_in != c.positions) {
    // separate records: what stays in place is copied (the moves write the filled slots later)
    const int n = cut ? keep : len;
    for (int j = tid; j < n; j += kEvictThreads) {
      c.weights[rec + j] = p.a.weights_in[rec + j];
      c.positions[rec + j] = p.a.positions_in[rec + j];
    }
  }
  if (!cut) {
    if (tid == 0) p.n_moves[row] = -1;
    return;
  }
  uint32_t prefix = 0;  // of the keep-th largest key
  int rest = keep;      // how many of the keys with this prefix stay
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < (1 << kRadixBits); i += kEvictThreads) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < len; j += kEvictThreads) {
      const uint32_t k = evict_key(p, rec, j, seen);
      if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1);
    }
    __syncthreads();
    // bins from the top: thread t takes the two bins below 2t from the top
    const int n = 1 << bits;
    int a0 = 0, a1 = 0;
    const int top = n - 1 - 2 * tid;
    if (top >= 1) {
      a0 = hist[top];
      a1 = hist[top - 1];
    }
    int total;
    const int before = block_scan(a0 + a1, s_warp, &total);
    if (top >= 1 && before < rest && before + a0 + a1 >= rest) {
      const bool second = before + a0 < rest;
      s_prefix = (prefix << bits) | static_cast<uint32_t>(second ? top - 1 : top);
      s_rest = rest - before - (second ? a0 : 0);
    }
    __syncthreads();
    prefix = s_prefix;
    rest = s_rest;
    __syncthreads();
  }
  // keys above the threshold stay, and the first `rest` slots whose key equals it
  int32_t* fill = p.moves + static_cast<int64_t>(row) * 2 * (c.max_slots / 2);
  int32_t* take = fill + c.max_slots / 2;
  int ties = 0, n_fill = 0, n_take = 0;
  for (int j0 = 0; j0 < len; j0 += kEvictThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < len ? evict_key(p, rec, j, seen) : 0u;
    int total;
    const int tie = j < len && k == prefix;
    const int order = ties + block_scan(tie, s_warp, &total);
    ties += total;
    const bool stays = j < len && (k > prefix || (tie && order < rest));
    const int f = j < keep && !stays, g = j >= keep && stays;
    int both;
    const int at = block_scan(f | (g << 16), s_warp, &both);
    if (f) fill[n_fill + (at & 0xffff)] = j;
    if (g) take[n_take + (at >> 16)] = j;
    n_fill += both & 0xffff;
    n_take += both >> 16;
  }
  if (tid == 0) p.n_moves[row] = n_fill;
}

// Moves rows: a warp per (slot to fill), keys then values, 16 bytes a lane where the layout
// allows it. Block (0, 0, b) sets the new length.
template <int kSize, bool kVec>
__global__ void __launch_bounds__(256) k_evict_move(const __grid_constant__ EvictParams p) {
  const KvView& c = p.c;
  const int kv = blockIdx.y, b = blockIdx.z, row = b * c.num_kv + kv;
  const int n = p.n_moves[row];
  if (kv == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    const int len = p.a.lens_in[b];
    c.lens[b] = n >= 0 ? p.a.keep : (len < 0 ? 0 : (len > c.max_slots ? c.max_slots : len));
  }
  const int32_t* fill = p.moves + static_cast<int64_t>(row) * 2 * (c.max_slots / 2);
  const int32_t* take = fill + c.max_slots / 2;
  const int lane = threadIdx.x & 31;
  const int64_t rec = static_cast<int64_t>(row) * c.max_slots;
  const int32_t* table = c.table + b * c.table_stride;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const int to = fill[i], from = take[i];
    const int64_t pt = table[to / c.page_size], pf = table[from / c.page_size];
    if (lane == 0) {
      c.weights[rec + to] = p.a.weights_in[rec + from];
      c.positions[rec + to] = p.a.positions_in[rec + from];
    }
    if (pt < 0 || pt >= c.num_pages || pf < 0 || pf >= c.num_pages) {
      if (lane == 0) atomicCAS(c.err, 0, kKvErrPage);
      continue;
    }
    const int st = to % c.page_size, sf = from % c.page_size;
    uint8_t* kt = c.k.base + (pt * c.k.page + st * c.k.slot + kv * c.k.head) * kSize;
    const uint8_t* kf = c.k.base + (pf * c.k.page + sf * c.k.slot + kv * c.k.head) * kSize;
    uint8_t* vt = c.v.base + (pt * c.v.page + st * c.v.slot + kv * c.v.head) * kSize;
    const uint8_t* vf = c.v.base + (pf * c.v.page + sf * c.v.slot + kv * c.v.head) * kSize;
    const int bytes = c.head_dim * kSize;
    if constexpr (kVec) {
      for (int o = 16 * lane; o < bytes; o += 512) {
        *reinterpret_cast<uint4*>(kt + o) = *reinterpret_cast<const uint4*>(kf + o);
        *reinterpret_cast<uint4*>(vt + o) = *reinterpret_cast<const uint4*>(vf + o);
      }
    } else {
      for (int o = lane; o < bytes; o += 32) {
        kt[o] = kf[o];
        vt[o] = vf[o];
      }
    }
  }
}

bool f32_aligned(const float* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0; }

} // namespace

KvCache::~KvCache() {
  cudaSetDevice(device);
  if (work) cudaFree(work);
}

static Status kv_alloc(KvCache* c) {
  KvView& v = c->view;
  WB_CUDA(cudaSetDevice(c->device));
  const size_t rows = static_cast<size_t>(v.num_seqs) * v.num_heads, heads = static_cast<size_t>(v.num_seqs) * v.num_kv;
  // one allocation, cut into the workspaces
  size_t bytes = 0;
  auto take = [&](size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  WB_TRY(attend_plan(c));
  const size_t err = take(4), ticket = take(4);
  const size_t part = take(c->part_bytes);  // from here on nothing needs to start as zero
  const size_t spans = take(c->span_bytes);
  const size_t scores = take(v.weights ? rows * v.max_slots * 4 : 0), lse = take(v.weights ? rows * 4 : 0);
  const size_t moves = take(v.positions ? heads * 2 * (v.max_slots / 2) * 4 : 0), n_moves = take(v.positions ? heads * 4 : 0);
  WB_CUDA(cudaMalloc(&c->work, bytes));
  c->err = reinterpret_cast<int*>(c->work + err);
  c->ticket = reinterpret_cast<int*>(c->work + ticket);
  c->spans = c->work + spans;
  c->part = reinterpret_cast<float*>(c->work + part);
  c->scores = reinterpret_cast<float*>(c->work + scores);
  c->lse = reinterpret_cast<float*>(c->work + lse);
  c->moves = reinterpret_cast<int32_t*>(c->work + moves);
  c->n_moves = reinterpret_cast<int32_t*>(c->work + n_moves);
  v.err = c->err;
  WB_CUDA(cudaMemset(c->work, 0, part));
  return cuda_status(cudaDeviceSynchronize(), "kv create");
}

Status kv_create(int device, KvType type, const KvView& view, KvCache** out) {
  auto* c = new KvCache();
  c->device = device;
  c->type = type;
  c->view = view;
  const Status st = kv_alloc(c);
  if (!st.ok()) {
    delete c;
    return st;
  }
  *out = c;
  return Status::Ok();
}

Status kv_append(KvCache* c, const KvAppendArgs& a, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(c->device));
  AppendParams p;
  p.a = a;
  p.c = c->view;
  if (!p.a.start) p.a.start = p.c.lens;
  if (!p.a.start_seen) p.a.start_seen = p.c.seen == p.c.lens ? p.a.start : p.c.seen;
  p.half = a.theta > 0.0 ? p.c.head_dim / 2 : 0;
  p.ticket = c->ticket;
  if (p.half > 0) {
    if (c->theta != a.theta) {
      c->inv_turns.resize(p.half);
      for (int i = 0; i < p.half; ++i)
        c->inv_turns[i] = std::pow(a.theta, -2.0 * i / p.c.head_dim) / 3.14159265358979323846;
      c->theta = a.theta;
    }
    for (int i = 0; i < p.half; ++i) p.rope.turns[i] = c->inv_turns[i];
  }
  const int size = kv_size(c->type);
  const bool vec = p.c.head_dim % 8 == 0 && pool_aligned(p.c.k, size, 4 * size) && pool_aligned(p.c.v, size, 4 * size) &&
                   f32_aligned(a.k, a.k_ld) && f32_aligned(a.v, a.v_ld) &&
                   (!a.q || (f32_aligned(a.q, a.q_ld) && f32_aligned(a.q_out, a.q_out_ld)));
  return by_type(c->type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int blocks = a.rows > 0 ? a.rows : 1;  // no row: the lengths are still carried over
    if (vec) k_append<T, true><<<blocks, kAppendThreads, 0, st>>>(p);
    else k_append<T, false><<<blocks, kAppendThreads, 0, st>>>(p);
    return cuda_status(cudaGetLastError(), "kv append launch");
  });
}

Status kv_evict(KvCache* c, const KvEvictArgs& a, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(c->device));
  EvictParams p;
  p.a = a;
  p.c = c->view;
  if (!p.a.lens_in) p.a.lens_in = p.c.lens;
  if (!p.a.weights_in) p.a.weights_in = p.c.weights;
  if (!p.a.positions_in) p.a.positions_in = p.c.positions;
  p.moves = c->moves;
  p.n_moves = c->n_moves;
  k_evict_select<<<dim3(p.c.num_kv, p.c.num_seqs), kEvictThreads, 0, st>>>(p);
  WB_TRY(cuda_status(cudaGetLastError(), "kv evict launch"));
  const int size = kv_size(c->type);
  const bool vec = p.c.head_dim * size % 16 == 0 && pool_aligned(p.c.k, size, 16) && pool_aligned(p.c.v, size, 16);
  int blocks = (p.c.max_slots / 2 + 7) / 8;
  if (blocks > 64) blocks = 64;
  if (blocks < 1) blocks = 1;
  const dim3 grid(blocks, p.c.num_kv, p.c.num_seqs);
  auto go = [&](auto size_c) {
    constexpr int S = decltype(size_c)::value;
    if (vec) k_evict_move<S, true><<<grid, 256, 0, st>>>(p);
    else k_evict_move<S, false><<<grid, 256, 0, st>>>(p);
  };
  if (size == 4) go(std::integral_constant<int, 4>{});
  else if (size == 2) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
  return cuda_status(cudaGetLastError(), "kv evict move launch");
}

Status kv_check_error(KvCache* c, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(c->device));
  int e = 0;
  WB_CUDA(cudaMemcpyAsync(&e, c->err, 4, cudaMemcpyDeviceToHost, st));
  WB_CUDA(cudaStreamSynchronize(st));
  if (e == 0) return Status::Ok();
  WB_CUDA(cudaMemsetAsync(c->err, 0, 4, st));
  WB_CUDA(cudaStreamSynchronize(st));
  if (e == kKvErrPage) return Status::Invalid("kv: a page id of the table is outside the pool");
  return Status::Invalid("kv: a length or an append is outside the sequence's slots");
}

} // namespace wb
