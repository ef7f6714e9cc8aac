// kvcache.cu -- append and eviction over a paged key-value cache, and its handle (sm_100a).
#include "kvcache.hpp"
#include "kvcache.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

namespace wb {
namespace {

// ---------------------------------------------------------------- append

// Rotary angles are position * theta^(-2i/D); the host passes them in half turns (angle / pi), whose
// cosine and sine are taken in 64 bits and rounded once: exact to 2^-25 at any position, which an
// angle of 32 bits would lose past position 10^3. (With the angle rounded to 32 bits after its whole
// turns were taken off, keys lay 1.26 times as far from 64 bits as the formula in fp32 does.)
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

// A pair's rotation as the formula has it in fp32, products rounded before they are added: what is
// stored is then what x0 * cos - x1 * sin gives anywhere, to the last code of an 8-bit page.
__device__ __forceinline__ void rotate(float& a, float& b, float cs, float sn) {
  const float x0 = a, x1 = b;
  a = __fsub_rn(__fmul_rn(x0, cs), __fmul_rn(x1, sn));
  b = __fadd_rn(__fmul_rn(x0, sn), __fmul_rn(x1, cs));
}

// One block per new token: the token's angles once into shared memory, then its key, value and
// query heads, pair (d, d + half) by pair. HBM bound: 4 B read per element, the page's type
// written (and 4 B for q). kVec: four consecutive pairs a thread (16-byte accesses).
// kDim: the width, 0 where it is not a constant (13k prompt tokens of 48 heads of 128: 81 us, 95 without).
// kDiv: the scales are not both powers of two (the same tokens: 100 us).
template <typename T, bool kVec, int kDim, bool kDiv>
__global__ void __launch_bounds__(kAppendThreads, 4) k_append(const __grid_constant__ AppendParams p) {
  __shared__ float s_cos[kMaxPairs], s_sin[kMaxPairs];
  __shared__ int s_last;
  const KvView& c = p.c;
  const int t = blockIdx.x, tid = threadIdx.x;
  const int D = kDim > 0 ? kDim : c.head_dim, half = p.half;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int kv_heads = c.num_kv, heads = 2 * kv_heads + (p.a.q ? c.num_heads : 0);
  auto source = [&](int h) {
    return h < kv_heads ? p.a.k + t * p.a.k_ld + static_cast<int64_t>(h) * D
                        : (h < 2 * kv_heads ? p.a.v + t * p.a.v_ld + static_cast<int64_t>(h - kv_heads) * D
                                            : p.a.q + t * p.a.q_ld + static_cast<int64_t>(h - 2 * kv_heads) * D);
  };
  // An item is four dims of a head's lower half and their partners; the first items' loads go out
  // before the row's place and angles are looked up.
  constexpr int kFly = 4;
  const int per = D / 8, h2 = D / 2, items = heads * per;
  float4 lo[kFly], hi[kFly];
  auto load = [&](int first) {
#pragma unroll
    for (int x = 0; x < kFly; ++x) {
      const int w = first + x * kAppendThreads;
      if (w >= items) continue;
      const int h = w / per;
      const float* src = source(h) + 4 * (w - h * per);
      lo[x] = *reinterpret_cast<const float4*>(src);
      hi[x] = *reinterpret_cast<const float4*>(src + h2);
    }
  };
  if constexpr (kVec) {
    if (t < p.a.rows) load(tid);
  }
  // the row's sequence: the last s with cu[s] <= t
  int seq = p.a.only >= 0 ? p.a.only : t, i = p.a.only >= 0 ? t : 0;
  bool live = t < p.a.rows;
  if (p.a.cu) {
    int a = 0, b = c.num_seqs;  // cu[a] <= t < cu[b] is what a row of a sequence has
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (p.a.cu[mid] <= t) a = mid; else b = mid;
    }
    seq = a;
    i = t - p.a.cu[seq];
    live = live && i >= 0 && i <= t && t < p.a.cu[seq + 1];
  } else if (p.a.active) {
    live = live && p.a.active[seq] != 0;
  } else if (p.a.only >= 0 && p.a.start[seq] != 0) {
    live = false;
    if (tid == 0) atomicCAS(c.err, 0, kKvErrHeld);
  }
  if (live) {
    const int64_t slot = static_cast<int64_t>(p.a.start[seq]) + i;
    const int64_t pos = static_cast<int64_t>(p.a.only >= 0 ? 0 : p.a.start_seen[seq]) + i;
    const bool in_range = slot >= 0 && slot < c.max_slots;
    const int at_page = in_range ? static_cast<int>(slot) / c.page_size : 0, in_page = in_range ? static_cast<int>(slot) - at_page * c.page_size : 0;
    int64_t page = in_range ? c.table[seq * c.table_stride + at_page] : -1;  // on its way while the angles are taken
    for (int d = tid; d < half; d += kAppendThreads) {
      double sn, cs;
      sincospi(static_cast<double>(pos) * p.rope.turns[d], &sn, &cs);
      s_sin[d] = static_cast<float>(sn);
      s_cos[d] = static_cast<float>(cs);
    }
    if (!in_range) {
      if (tid == 0) atomicCAS(c.err, 0, kKvErrSlot);
    } else if (page < 0 || page >= c.num_pages) {
      page = -1;
      if (tid == 0) atomicCAS(c.err, 0, kKvErrPage);
    }
    __syncthreads();
    T* kd = reinterpret_cast<T*>(c.k.base) + page * c.k.page + in_page * c.k.slot;
    T* vd = reinterpret_cast<T*>(c.v.base) + page * c.v.page + in_page * c.v.slot;
    const float ks = 1.0f / c.k_scale, vs = 1.0f / c.v_scale;
    float* qo = p.a.q_out + t * p.a.q_out_ld;
    if constexpr (kVec) {
      for (int first = tid; first < items; first += kFly * kAppendThreads) {
        if (first != tid) load(first);
#pragma unroll
        for (int x = 0; x < kFly; ++x) {
          const int w = first + x * kAppendThreads;
          if (w >= items) continue;
          const int h = w / per, d = 4 * (w - h * per);
          const bool is_v = h >= kv_heads && h < 2 * kv_heads;
          float a[4] = {lo[x].x, lo[x].y, lo[x].z, lo[x].w}, b[4] = {hi[x].x, hi[x].y, hi[x].z, hi[x].w};
          if (!is_v && half > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) rotate(a[e], b[e], s_cos[d + e], s_sin[d + e]);
          }
          if (h >= 2 * kv_heads) {
            float* o = qo + static_cast<int64_t>(h - 2 * kv_heads) * D;
            *reinterpret_cast<float4*>(o + d) = make_float4(a[0], a[1], a[2], a[3]);
            *reinterpret_cast<float4*>(o + d + h2) = make_float4(b[0], b[1], b[2], b[3]);
          } else if (page >= 0) {
            T* o = is_v ? vd + (h - kv_heads) * c.v.head : kd + h * c.k.head;
            const float scale = kDiv ? (is_v ? c.v_scale : c.k_scale) : 0.0f, inv = kDiv ? 0.0f : (is_v ? vs : ks);
            store4<T, kDiv>(o + d, a, scale, inv);
            store4<T, kDiv>(o + d + h2, b, scale, inv);
          }
        }
      }
    } else {
      // a pair of dims (d, d + n / 2) a thread, so that q may be rotated in place
      const int pairs = (D + 1) / 2;
      for (int w = tid; w < heads * pairs; w += kAppendThreads) {
        const int h = w / pairs, d0 = w - h * pairs, d1 = d0 + D / 2;
        const bool is_v = h >= kv_heads && h < 2 * kv_heads;
        const bool odd = d0 == D / 2;  // the unpaired last dim of an odd width
        const float* src = source(h);
        float a = odd ? 0.0f : src[d0], b = odd ? src[D - 1] : src[d1];
        if (!is_v && half > 0 && !odd) rotate(a, b, s_cos[d0], s_sin[d0]);
        const int db = odd ? D - 1 : d1;
        if (h >= 2 * kv_heads) {
          float* o = qo + static_cast<int64_t>(h - 2 * kv_heads) * D;
          if (!odd) o[d0] = a;
          o[db] = b;
        } else if (page >= 0) {
          T* o = is_v ? vd + (h - kv_heads) * c.v.head : kd + h * c.k.head;
          const float scale = kDiv ? (is_v ? c.v_scale : c.k_scale) : 0.0f, inv = kDiv ? 0.0f : (is_v ? vs : ks);
          if (!odd) o[d0] = to_stored<T>(over<kDiv>(a, scale, inv));
          o[db] = to_stored<T>(over<kDiv>(b, scale, inv));
        }
      }
    }
    if (in_range) {
      for (int h = tid; h < kv_heads; h += kAppendThreads) {
        const int64_t at = (static_cast<int64_t>(seq) * kv_heads + h) * c.max_slots + slot;
        if (c.positions) c.positions[at] = static_cast<int32_t>(pos);
        if (c.weights) c.weights[at] = 0.0f;
      }
    }
  }
  // The last block to finish advances the lengths: start may be lens itself, which every thread of
  // every block has read by then.
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) *p.ticket = 0;
  for (int s = tid; s < c.num_seqs; s += kAppendThreads) {
    if (p.a.active && p.a.active[s] == 0) {
      p.a.step_lens[s] = 0;
      continue;
    }
    if (p.a.only >= 0 && (s != p.a.only || p.a.start[s] != 0)) continue;
    int64_t n = p.a.only < 0 ? 1 : p.a.rows;
    if (p.a.cu) {  // the rows that there are
      const int64_t from = p.a.cu[s], to = p.a.cu[s + 1];
      n = from < 0 ? 0 : max(min(to, static_cast<int64_t>(p.a.rows)) - from, static_cast<int64_t>(0));
      if (n != to - from) atomicCAS(c.err, 0, kKvErrRows);
    }
    const int64_t len = static_cast<int64_t>(p.a.start[s]) + n, tot = static_cast<int64_t>(p.a.only >= 0 ? 0 : p.a.start_seen[s]) + n;
    c.lens[s] = static_cast<int32_t>(len < c.max_slots ? len : c.max_slots);
    if (p.a.active) p.a.step_lens[s] = c.lens[s];
    if (c.seen != c.lens) c.seen[s] = static_cast<int32_t>(tot);
  }
}

// ---------------------------------------------------------------- eviction

struct EvictParams {
  KvEvictArgs a;
  KvView c;
  int32_t* moves;    // [num_seqs][num_kv][2][max_slots / 2]: slots to fill, slots to take
  int32_t* n_moves;  // [num_seqs][num_kv]; -1: not cut
  int* tickets;      // [num_seqs], zero between calls
  int cached;        // keys a block keeps in shared memory (0: read again in each pass)
};

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kMaxRanks = 8;          // blocks of a cluster
constexpr int kRadixBins = 2048;      // three passes over a 32-bit key: 11 + 11 + 10 bits
constexpr int kEvictCache = 24 * 1024;  // keys: 96 KB

// The order in which slots stay: protected ones first, then by weight; larger keys stay. NaN counts
// as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int sinks, int recent_from) {
  if (pos < sinks || pos >= recent_from) return 0xffffffffu;
  if (isnan(w)) return 0x007fffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Rows of one (sequence, key-value head): slots `take` to slots `fill`, 16 bytes a lane where the
// layout allows it. A group of lanes takes a row; the next row's place is looked up while this
// one's values are on their way. Rows lie in random order, and a narrow one is a short access: of 24
// E4M3 heads of 128 cut from 40k..65k slots to 16k the move takes 32 us at about 3.5 TB/s of read and
// written rows (38 us with the look-up in line).
template <int kSize, bool kVec>
__device__ __forceinline__ void move_rows(const EvictParams& p, int b, int kv, const int32_t* fill, const int32_t* take,
                                          int n, int worker, int workers) {
  const KvView& c = p.c;
  const int64_t rec = (static_cast<int64_t>(b) * c.num_kv + kv) * c.max_slots;
  const int32_t* table = c.table + b * c.table_stride;
  const int lane = threadIdx.x & 31;
  const int bytes = c.head_dim * kSize;
  auto row_of = [&](int slot, int64_t* k, int64_t* v) {
    const int page_at = slot / c.page_size, in = slot - page_at * c.page_size;
    const int page = table[page_at];
    if (page < 0 || page >= c.num_pages) return false;
    *k = (page * c.k.page + in * c.k.slot + kv * c.k.head) * kSize;
    *v = (page * c.v.page + in * c.v.slot + kv * c.v.head) * kSize;
    return true;
  };
  if constexpr (kVec) {
    const int lanes = bytes > 256 ? 32 : (bytes > 128 ? 16 : 8);  // of a row
    const int groups = 32 / lanes, at = 16 * (lane % lanes), step = workers * groups;
    struct Row {  // slots and pages
      int to, from, to_page, to_in, from_page, from_in;
    };
    auto fetch = [&](int i) {
      Row r;
      r.to = fill[i];
      r.from = take[i];
      const int pt = r.to / c.page_size, pf = r.from / c.page_size;
      r.to_in = r.to - pt * c.page_size;
      r.from_in = r.from - pf * c.page_size;
      r.to_page = table[pt];
      r.from_page = table[pf];
      return r;
    };
    auto address = [&](const KvPool& q, int page, int in) { return q.base + (page * q.page + in * q.slot + kv * q.head) * kSize + at; };
    int i = worker * groups + lane / lanes;
    Row row{};
    if (i < n) row = fetch(i);
    for (; i < n; i += step) {
      uint4 k{}, v{};
      float weight = 0.0f;
      int pos = 0;
      if (at == 0) {
        weight = p.a.weights_in[rec + row.from];
        pos = p.a.positions_in[rec + row.from];
      }
      const bool ok = row.to_page >= 0 && row.to_page < c.num_pages && row.from_page >= 0 && row.from_page < c.num_pages;
      if (!ok) atomicCAS(c.err, 0, kKvErrPage);
      const uint8_t* const kf = address(c.k, row.from_page, row.from_in);
      const uint8_t* const vf = address(c.v, row.from_page, row.from_in);
      if (ok && at < bytes) {
        k = *reinterpret_cast<const uint4*>(kf);
        v = *reinterpret_cast<const uint4*>(vf);
      }
      Row ahead{};
      if (i + step < n) ahead = fetch(i + step);
      if (ok && at == 0) {
        c.weights[rec + row.to] = weight;
        c.positions[rec + row.to] = pos;
      }
      if (ok && at < bytes) {
        uint8_t* const kt = address(c.k, row.to_page, row.to_in);
        uint8_t* const vt = address(c.v, row.to_page, row.to_in);
        *reinterpret_cast<uint4*>(kt) = k;
        *reinterpret_cast<uint4*>(vt) = v;
        for (int o = 16 * lanes; at + o < bytes; o += 16 * lanes) {
          *reinterpret_cast<uint4*>(kt + o) = *reinterpret_cast<const uint4*>(kf + o);
          *reinterpret_cast<uint4*>(vt + o) = *reinterpret_cast<const uint4*>(vf + o);
        }
      }
      row = ahead;
    }
  } else {
    for (int i = worker; i < n; i += workers) {
      const int to = fill[i], from = take[i];
      int64_t kt, vt, kf, vf;
      if (!(row_of(to, &kt, &vt) && row_of(from, &kf, &vf))) {
        if (lane == 0) atomicCAS(c.err, 0, kKvErrPage);
        continue;
      }
      if (lane == 0) {
        c.weights[rec + to] = p.a.weights_in[rec + from];
        c.positions[rec + to] = p.a.positions_in[rec + from];
      }
      for (int o = lane; o < bytes; o += 32) {
        c.k.base[kt + o] = c.k.base[kf + o];
        c.v.base[vt + o] = c.v.base[vf + o];
      }
    }
  }
}

// A cluster of blocks per (sequence, key-value head), each with its share of the slots: the keep-th
// largest key by radix selection (histograms added over the cluster through distributed shared
// memory), then, in slot order, the slots below keep that go (to fill) and those above it that stay
// (to take). Both lists are equally long and no slot is in both, so the rows can move in any order.
// A cluster of one block moves them itself; larger ones leave the lists to k_evict_move.
// Latency bound: 8 bytes a slot are read, the rest is a dozen barriers. About 24 us of the 58
// at 24 heads of 40k..65k slots (10 MB read, eight blocks a head); 32 sequences x 8 heads of 1025..1056
// slots cut to 1024 take 10.4 us with their rows, in one launch.
template <int kSize, bool kVec>
__global__ void __launch_bounds__(kEvictThreads, 2) k_evict_select(const __grid_constant__ EvictParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ uint32_t s_keys[];
  __shared__ __align__(16) int s_hist[3][kRadixBins];
  __shared__ int s_group[3][kRadixBins / 32];
  __shared__ int s_warp[kEvictWarps], s_warp2[kEvictWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_rest, s_same;
  __shared__ int s_ties;      // of this block
  __shared__ int s_lists[2];  // slots of this block to fill, to take
  const KvView& c = p.c;
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int kv = blockIdx.x / ranks, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int row = b * c.num_kv + kv;
  const int64_t rec = static_cast<int64_t>(row) * c.max_slots;
  asm volatile("griddepcontrol.launch_dependents;");
  for (int i = tid; i < 3 * kRadixBins; i += kEvictThreads) (&s_hist[0][0])[i] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int given = p.a.lens_in[b], keep = p.a.keep, recent_from = c.seen[b] - p.a.recent;
  const int len = min(max(given, 0), c.max_slots);
  if (len != given && tid == 0) atomicCAS(c.err, 0, kKvErrSlot);
  const bool cut = len > p.a.budget;
  // this block's slots, and each warp's: multiples of 32
  const int per = ((len + ranks - 1) / ranks + 31) & ~31;
  const int lo = min(rank * per, len), hi = min(lo + per, len);
  const int per_warp = (((hi - lo) + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
  const int wlo = min(lo + w * per_warp, hi), whi = min(wlo + per_warp, hi);
  const bool apart = p.a.weights_in != c.weights || p.a.positions_in != c.positions;
  const int stays_to = cut ? keep : len;  // separate records: what stays in place is copied
  auto key_at = [&](int j) -> uint32_t {
    if (p.cached) return s_keys[j - lo];
    return evict_key(p.a.weights_in[rec + j], p.a.positions_in[rec + j], p.a.sinks, recent_from);
  };
  if (cut || apart) {
    constexpr int kFly = 8;  // slots whose loads are in flight together (the stores may alias them)
    for (int j0 = lo + tid; j0 < hi; j0 += kFly * kEvictThreads) {
      float weight[kFly];
      int pos[kFly];
#pragma unroll
      for (int x = 0; x < kFly; ++x) {
        const int j = j0 + x * kEvictThreads;
        weight[x] = j < hi ? p.a.weights_in[rec + j] : 0.0f;
        pos[x] = j < hi ? p.a.positions_in[rec + j] : 0;
      }
#pragma unroll
      for (int x = 0; x < kFly; ++x) {
        const int j = j0 + x * kEvictThreads;
        if (j >= hi) break;
        if (apart && j < stays_to) {
          c.weights[rec + j] = weight[x];
          c.positions[rec + j] = pos[x];
        }
        if (cut && p.cached) s_keys[j - lo] = evict_key(weight[x], pos[x], p.a.sinks, recent_from);
      }
    }
  }
  // The last (head, block) of a sequence to have read its length writes the new one.
  auto leave = [&] {
    if (tid == 0 && atomicAdd(p.tickets + b, 1) == c.num_kv * ranks - 1) {
      p.tickets[b] = 0;
      c.lens[b] = stays_to;
    }
  };
  if (!cut) {
    if (rank == 0 && tid == 0) p.n_moves[row] = -1;
    leave();
    return;  // the whole cluster does
  }
  __syncthreads();


  uint32_t prefix = 0;  // of the keep-th largest key
  int rest = keep;      // how many of the keys with this prefix stay
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bits = pass == 2 ? 10 : 11;
    int* hist = s_hist[pass];
    for (int j = lo + tid; j < hi; j += kEvictThreads) {
      const uint32_t k = key_at(j);
      if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1);
    }
    // sums of 32 bins each, then one warp finds the group and the bin, adding over the cluster
    __syncthreads();
    const int4 four = *reinterpret_cast<const int4*>(hist + 4 * tid);
    int sum = four.x + four.y + four.z + four.w;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((lane & 7) == 0) s_group[pass][tid >> 3] = sum;
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    if (w == 0) {
      auto total = [&](const int* at) {  // of one counter over the cluster
        int q[kMaxRanks];
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r) q[r] = r < ranks ? *(ranks > 1 ? cluster.map_shared_rank(at, r) : at) : 0;
        int n = 0;
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r) n += q[r];
        return n;
      };
      // lane i holds n, the i-th from the top; the lane in which `left` is used up
      auto find = [&](int n, int& left) {
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        const int at = __ffs(__ballot_sync(0xffffffffu, x >= left)) - 1;
        left -= __shfl_sync(0xffffffffu, x - n, at);
        return at;
      };
      int left = rest;
      const int upper = total(&s_group[pass][kRadixBins / 32 - 1 - 2 * lane]), lower = total(&s_group[pass][kRadixBins / 32 - 2 - 2 * lane]);
      const int pair = find(upper + lower, left);
      const int in_upper = __shfl_sync(0xffffffffu, upper, pair);
      int group = kRadixBins / 32 - 1 - 2 * pair;
      if (left > in_upper) {
        left -= in_upper;
        --group;
      }
      const int n = total(hist + 32 * group + 31 - lane);
      const int bin = find(n, left);
      const int same = __shfl_sync(0xffffffffu, n, bin);
      if (lane == 0) {
        s_prefix = (prefix << bits) | static_cast<uint32_t>(32 * group + 31 - bin);
        s_rest = left;
        s_same = same;
      }
    }
    __syncthreads();
    prefix = s_prefix;
    rest = s_rest;
    __syncthreads();
  }

  // Keys above the threshold stay, and the first `rest` slots whose key equals it; where all of those
  // stay (no ties but within the kept), their order is not needed.
  int ties_before = 0;
  if (s_same != rest) {
    int ties = 0;
    for (int j0 = wlo; j0 < whi; j0 += 32) ties += __popc(__ballot_sync(0xffffffffu, j0 + lane < whi && key_at(min(j0 + lane, whi - 1)) == prefix));
    if (lane == 0) s_warp[w] = ties;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < kEvictWarps; ++i) {
      if (i < w) ties_before += s_warp[i];
      all += s_warp[i];
    }
    if (tid == 0) s_ties = all;
    if (ranks > 1) {
      cluster.sync();
      int t[kMaxRanks];
#pragma unroll
      for (int r = 0; r < kMaxRanks; ++r) t[r] = r < rank ? *cluster.map_shared_rank(&s_ties, r) : 0;
#pragma unroll
      for (int r = 0; r < kMaxRanks; ++r) ties_before += t[r];
    }
    __syncthreads();
  }
  auto flags_at = [&](int j0, int& seen_ties, uint32_t& f, uint32_t& g) {
    const int j = j0 + lane;
    const uint32_t k = j < whi ? key_at(j) : 0u;
    const uint32_t tie = __ballot_sync(0xffffffffu, j < whi && k == prefix);
    const int order = seen_ties + __popc(tie & ((1u << lane) - 1u));
    const bool stays = j < whi && (k > prefix || (k == prefix && order < rest));
    f = __ballot_sync(0xffffffffu, j < whi && j < keep && !stays);
    g = __ballot_sync(0xffffffffu, j >= keep && stays);
    seen_ties += __popc(tie);
  };
  int n_fill = 0, n_take = 0, seen_ties = ties_before;
  for (int j0 = wlo; j0 < whi; j0 += 32) {
    uint32_t f, g;
    flags_at(j0, seen_ties, f, g);
    if (p.cached && lane == 0) {  // kept where the warp's keys were
      s_keys[j0 - lo] = f;
      s_keys[j0 - lo + 1] = g;
    }
    n_fill += __popc(f);
    n_take += __popc(g);
  }
  __syncthreads();
  if (lane == 0) {
    s_warp[w] = n_fill;
    s_warp2[w] = n_take;
  }
  __syncthreads();
  int fill_at = 0, take_at = 0, fills = 0, takes = 0;
#pragma unroll
  for (int i = 0; i < kEvictWarps; ++i) {
    if (i < w) {
      fill_at += s_warp[i];
      take_at += s_warp2[i];
    }
    fills += s_warp[i];
    takes += s_warp2[i];
  }
  if (tid == 0) {
    s_lists[0] = fills;
    s_lists[1] = takes;
  }
  int moved = fills;
  if (ranks > 1) {
    cluster.sync();
    moved = 0;
    int f[kMaxRanks], g[kMaxRanks];
#pragma unroll
    for (int r = 0; r < kMaxRanks; ++r) {
      f[r] = g[r] = 0;
      if (r < ranks) {
        const int* l = cluster.map_shared_rank(s_lists, r);
        f[r] = l[0];
        g[r] = l[1];
      }
    }
#pragma unroll
    for (int r = 0; r < kMaxRanks; ++r) {
      if (r < rank) {
        fill_at += f[r];
        take_at += g[r];
      }
      moved += f[r];
    }
  }
  int32_t* fill = p.moves + static_cast<int64_t>(row) * 2 * (c.max_slots / 2);
  int32_t* take = fill + c.max_slots / 2;
  seen_ties = ties_before;
  for (int j0 = wlo; j0 < whi; j0 += 32) {
    uint32_t f, g;
    if (p.cached) {
      f = s_keys[j0 - lo];
      g = s_keys[j0 - lo + 1];
    } else {
      flags_at(j0, seen_ties, f, g);
    }
    const uint32_t below = (1u << lane) - 1u;
    if ((f >> lane) & 1) fill[fill_at + __popc(f & below)] = j0 + lane;
    if ((g >> lane) & 1) take[take_at + __popc(g & below)] = j0 + lane;
    fill_at += __popc(f);
    take_at += __popc(g);
  }
  if (ranks == 1) {
    __syncthreads();  // the block's own lists
    move_rows<kSize, kVec>(p, b, kv, fill, take, moved, w, kEvictWarps);
  } else {
    if (rank == 0 && tid == 0) p.n_moves[row] = moved;
    cluster.sync();  // no block leaves while another reads its shared memory
  }
  leave();
}

template <int kSize, bool kVec>
__global__ void __launch_bounds__(256, 4) k_evict_move(const __grid_constant__ EvictParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const KvView& c = p.c;
  const int kv = blockIdx.y, b = blockIdx.z, row = b * c.num_kv + kv;
  const int32_t* fill = p.moves + static_cast<int64_t>(row) * 2 * (c.max_slots / 2);
  move_rows<kSize, kVec>(p, b, kv, fill, fill + c.max_slots / 2, p.n_moves[row], blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8);
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
  const size_t err = take(4), ticket = take(4), step_lens = take(static_cast<size_t>(v.num_seqs) * 4);
  const size_t evict_tickets = take(v.positions ? static_cast<size_t>(v.num_seqs) * 4 : 0);
  const size_t part = take(c->part_bytes);  // from here on nothing needs to start as zero
  const size_t spans = take(c->span_bytes);
  const size_t scores = take(v.weights ? rows * v.max_slots * 4 : 0), lse = take(v.weights ? rows * 4 : 0);
  const size_t moves = take(v.positions ? heads * 2 * (v.max_slots / 2) * 4 : 0), n_moves = take(v.positions ? heads * 4 : 0);
  WB_CUDA(cudaMalloc(&c->work, bytes));
  c->err = reinterpret_cast<int*>(c->work + err);
  c->ticket = reinterpret_cast<int*>(c->work + ticket);
  c->step_lens = reinterpret_cast<int32_t*>(c->work + step_lens);
  c->evict_tickets = reinterpret_cast<int*>(c->work + evict_tickets);
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
    cudaGetLastError();  // a failed allocation must not be taken for a later launch's error
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
    // both reciprocals exact: the fraction of a power of two is one half
    int e;
    const bool exact = std::frexp(p.c.k_scale, &e) == 0.5f && std::frexp(p.c.v_scale, &e) == 0.5f;
    auto* kernel = !vec ? (exact ? k_append<T, false, 0, false> : k_append<T, false, 0, true>)
                        : (!exact ? k_append<T, true, 0, true>
                                  : (p.c.head_dim == 128 ? k_append<T, true, 128, false>
                                                         : (p.c.head_dim == 64 ? k_append<T, true, 64, false> : k_append<T, true, 0, false>)));
    return launch_after(kernel, dim3(blocks), kAppendThreads, 0, st, p);
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
  p.tickets = c->evict_tickets;
  const int size = kv_size(c->type);
  const bool vec = p.c.head_dim * size % 16 == 0 && pool_aligned(p.c.k, size, 16) && pool_aligned(p.c.v, size, 16);
  // One block a head unless that leaves SMs idle or a block's keys do not fit its shared memory.
  const int64_t heads = static_cast<int64_t>(p.c.num_seqs) * p.c.num_kv;
  int ranks = 1;
  while (ranks < kMaxRanks && ((heads * ranks < 148 && p.c.max_slots / ranks > 2048) || p.c.max_slots / ranks > kEvictCache - 32)) ranks *= 2;
  const int per = ((p.c.max_slots + ranks - 1) / ranks + 31) & ~31;
  p.cached = per <= kEvictCache;
  auto go = [&](auto size_c, auto vec_c) -> Status {
    constexpr int S = decltype(size_c)::value;
    constexpr bool V = decltype(vec_c)::value;
    auto* select = k_evict_select<S, V>;
    WB_CUDA(cudaFuncSetAttribute(select, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictCache * 4));
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {static_cast<unsigned>(ranks), 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.c.num_kv * ranks, p.c.num_seqs);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = p.cached ? per * 4 : 0;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    WB_TRY(cuda_status(cudaLaunchKernelEx(&cfg, select, p), "kv evict launch"));
    if (ranks == 1) return Status::Ok();
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>((p.c.max_slots / 2 + 63) / 64, std::max<int64_t>(1, 148 * 8 / heads))),
                       p.c.num_kv, p.c.num_seqs);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, k_evict_move<S, V>, p), "kv evict move launch");
  };
  auto by_size = [&](auto vec_c) -> Status {
    if (size == 4) return go(std::integral_constant<int, 4>{}, vec_c);
    if (size == 2) return go(std::integral_constant<int, 2>{}, vec_c);
    return go(std::integral_constant<int, 1>{}, vec_c);
  };
  return vec ? by_size(std::true_type{}) : by_size(std::false_type{});
}

Status kv_check_error(KvCache* c, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(c->device));
  int e = 0;
  WB_CUDA(cudaMemcpyAsync(&e, c->err, 4, cudaMemcpyDeviceToHost, st));
  WB_CUDA(cudaStreamSynchronize(st));
  if (e == 0) return Status::Ok();
  WB_CUDA(cudaMemsetAsync(c->err, 0, 4, st));
  WB_CUDA(cudaStreamSynchronize(st));
  if (e == kKvErrRows) return Status::Invalid("kv append: cu_tokens decreases, is negative or goes past the rows");
  if (e == kKvErrHeld) return Status::Invalid("kv: a prompt for a sequence that holds slots already");
  if (e == kKvErrPage) return Status::Invalid("kv: a page id of the table is outside the pool");
  return Status::Invalid("kv: a length or an append is outside the sequence's slots");
}

} // namespace wb
