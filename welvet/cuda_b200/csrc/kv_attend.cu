// kv_attend.cu -- attention of one new token per sequence over a paged key-value cache (sm_100a).
//
// z_j = scale q.k_j - slope (p_q - p_j), w = softmax(z), o = sum_j w_j v_j, in one pass over the
// keys with a running maximum and sum; all scores are held in units of log2, so that a weight is
// one exp2. HBM bound: a key and a value row are read once for all the query heads that share
// them, 2 sizeof(T) head_dim bytes against 4 head_dim flops per query head. Measured, 8 key-value
// heads of 128, 4 query heads each: 64 sequences of 8191 slots (2.15 GB), bf16 351 to 372 us by the GPU
// and its power cap, 5.8 to 6.1 TB/s (88 to 93 % of a copy), f16 340 us, 6.3 TB/s; f32, 16 sequences of
// 8191 (1.07 GB), 240 to 247 us, 4.4 TB/s: four MMAs and eight conversions of parts a step bound it;
// E4M3, 30k..131k slots (0.87 GB), 177 to 182 us, 4.9 TB/s: half the bytes of bf16 for the same products,
// so instruction issue and its latency at 8 warps an SM bound it before the copies do.
#include "kvcache.cuh"
#include "kvcache.hpp"
#include "pipeline.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

namespace wb {
namespace {

constexpr int kMaxCluster = 8;  // blocks of a cluster
constexpr float kLog2e = 1.4426950408889634f;

struct KvBytes {  // a pool's strides in bytes
  uint32_t page, slot, head;
};

struct AttendParams {
  KvAttendArgs a;
  KvView c;
  KvBytes kb, vb;  // tiled form
  int same;        // the two pools have the same strides
  int splits;      // simple form
  float* part;     // partial results: o, m, l
  float* scores;   // with accumulate: [num_seqs][num_heads][max_slots], units of log2
  float* lse;      // [num_seqs][num_heads]
  // tiled form
  int group;       // query heads per key-value head
  int head_groups; // of eight query heads of a key-value head
  int page_shift;  // log2(page_size), or -1
  int cluster;     // blocks of a unit that join through distributed shared memory (0: runs)
  int2* spans;     // [num_seqs][num_kv]: first run and number of runs of a unit
};

// ---------------------------------------------------------------- one query head a block

constexpr int kSimpleWarps = 4;
constexpr int kSimpleDims = 8;  // dims a lane holds: head_dim <= 256

// The form for layouts that 16-byte copies cannot serve (rows off 16-byte boundaries, a head_dim
// that is no multiple of 8 elements). A block takes one split of one (sequence, query head); a warp
// a key at a time, lanes over the head's dims, one pass with the running maximum and sum. Keys
// shared by the heads of a group are read again for each head.
template <typename T>
__global__ void __launch_bounds__(32 * kSimpleWarps) k_attend_simple(const __grid_constant__ AttendParams p) {
  __shared__ float s_m[kSimpleWarps], s_l[kSimpleWarps];
  __shared__ float s_o[kSimpleWarps][32 * kSimpleDims];
  const KvView& c = p.c;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int D = c.head_dim, kv = h / (c.num_heads / c.num_kv);
  int len = c.lens[b];
  if (len < 0 || len > c.max_slots) {
    if (threadIdx.x == 0) atomicCAS(c.err, 0, kKvErrSlot);
    len = len < 0 ? 0 : c.max_slots;
  }
  const int64_t per = (len + p.splits - 1) / p.splits;
  const int j0 = static_cast<int>(per * split < len ? per * split : len);
  const int j1 = static_cast<int>(per * (split + 1) < len ? per * (split + 1) : len);
  const int q_pos = c.positions ? c.seen[b] - 1 : len - 1;
  const int64_t rec = (static_cast<int64_t>(b) * c.num_kv + kv) * c.max_slots;
  const float slope = p.a.alibi ? alibi_slope(h, c.num_heads) * kLog2e : 0.0f;
  float q[kSimpleDims], o[kSimpleDims];
#pragma unroll
  for (int i = 0; i < kSimpleDims; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < D ? p.a.q[b * p.a.q_ld + static_cast<int64_t>(h) * D + d] * (p.a.scale * c.k_scale * kLog2e) : 0.0f;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j = j0 + w; j < j1; j += kSimpleWarps) {
    const int pos = c.positions ? c.positions[rec + j] : j;
    const int page = c.table[b * c.table_stride + j / c.page_size];
    bool ok = page >= 0 && page < c.num_pages;
    if (!ok && lane == 0) atomicCAS(c.err, 0, kKvErrPage);
    if (p.a.window > 0 && pos <= q_pos - p.a.window) ok = false;
    float z = -INFINITY;
    if (ok) {
      const T* kr = reinterpret_cast<const T*>(c.k.base) + page * c.k.page + (j % c.page_size) * c.k.slot + kv * c.k.head;
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < kSimpleDims; ++i) {
        const int d = lane + 32 * i;
        if (d < D) dot += q[i] * to_float(kr[d]);
      }
      z = warp_sum(dot) - slope * static_cast<float>(q_pos - pos);
      const T* vr = reinterpret_cast<const T*>(c.v.base) + page * c.v.page + (j % c.page_size) * c.v.slot + kv * c.v.head;
      const float m_new = fmaxf(m, z);
      const float ref = m_new == -INFINITY ? 0.0f : m_new;
      const float e = exp2f(z - ref), corr = exp2f(m - ref);
      l = l * corr + e;
#pragma unroll
      for (int i = 0; i < kSimpleDims; ++i) {
        const int d = lane + 32 * i;
        if (d < D) o[i] = o[i] * corr + e * to_float(vr[d]);
      }
      m = m_new;
    }
    if (p.a.accumulate && lane == 0)
      p.scores[(static_cast<int64_t>(b) * c.num_heads + h) * c.max_slots + j] = ok ? z : -INFINITY;
  }
  if (lane == 0) {
    s_m[w] = m;
    s_l[w] = l;
  }
#pragma unroll
  for (int i = 0; i < kSimpleDims; ++i) s_o[w][lane + 32 * i] = o[i];
  __syncthreads();
  float mm = s_m[0];
#pragma unroll
  for (int i = 1; i < kSimpleWarps; ++i) mm = fmaxf(mm, s_m[i]);
  const float ref = mm == -INFINITY ? 0.0f : mm;
  float* dst = p.part + ((static_cast<int64_t>(b) * c.num_heads + h) * p.splits + split) * (D + 2);
  for (int d = threadIdx.x; d < D; d += 32 * kSimpleWarps) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kSimpleWarps; ++i) v += s_o[i][d] * exp2f(s_m[i] - ref);
    dst[d] = v;
  }
  if (threadIdx.x == 0) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kSimpleWarps; ++i) v += s_l[i] * exp2f(s_m[i] - ref);
    dst[D] = mm;
    dst[D + 1] = v;
  }
}

// Joins the splits of one (sequence, query head) in split order. A row that nothing is allowed
// in has l = 0 and m = -inf from every split: its output is zero.
__global__ void k_attend_join(const __grid_constant__ AttendParams p) {
  const KvView& c = p.c;
  const int h = blockIdx.x, b = blockIdx.y, D = c.head_dim;
  const float* src = p.part + (static_cast<int64_t>(b) * c.num_heads + h) * p.splits * (D + 2);
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, src[s * (D + 2) + D]);
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int s = 0; s < p.splits; ++s) l += src[s * (D + 2) + D + 1] * exp2f(src[s * (D + 2) + D] - ref);
  const float inv = l == 0.0f ? 0.0f : c.v_scale / l;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float v = 0.0f;
    for (int s = 0; s < p.splits; ++s) v += src[s * (D + 2) + d] * exp2f(src[s * (D + 2) + D] - ref);
    p.a.out[b * p.a.out_ld + static_cast<int64_t>(h) * D + d] = v * inv;
  }
  if (threadIdx.x == 0 && p.a.accumulate) p.lse[static_cast<int64_t>(b) * c.num_heads + h] = l == 0.0f ? INFINITY : ref + log2f(l);
}

// weights[j] = weights_in[j] + sum over the group's heads of 2^(score - lse), heads in order, for
// every step-th slot from `first`. The first slots' loads go out before `ready` (which makes lse).
template <typename F>
__device__ __forceinline__ void add_weights(const AttendParams& p, int b, int kv, const float* lse, int first, int step, F&& ready) {
  const KvView& c = p.c;
  const int group = c.num_heads / c.num_kv;
  int len = c.lens[b];
  len = len < 0 ? 0 : (len > c.max_slots ? c.max_slots : len);
  const int lo = p.a.window > 0 && !c.positions ? len - p.a.window : 0;  // slots below have no score
  const int64_t rec = (static_cast<int64_t>(b) * c.num_kv + kv) * c.max_slots;
  const float* scores = p.scores + (static_cast<int64_t>(b) * c.num_heads + kv * group) * c.max_slots;
  constexpr int kFly = 4, kHeads = 4;  // slots and heads in flight together
  float s[kFly], z[kHeads][kFly];
  auto load = [&](int j0, int i0) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
#pragma unroll
      for (int x = 0; x < kFly; ++x) {
        const int j = j0 + x * step;
        z[i][x] = i0 + i < group && j >= lo && j < len ? scores[static_cast<int64_t>(i0 + i) * c.max_slots + j] : -INFINITY;
      }
  };
  auto start = [&](int j0) {
#pragma unroll
    for (int x = 0; x < kFly; ++x) s[x] = j0 + x * step < len ? p.a.weights_in[rec + j0 + x * step] : 0.0f;
    load(j0, 0);
  };
  if (first < len) start(first);
  ready();
  for (int j0 = first; j0 < len; j0 += kFly * step) {
    if (j0 != first) start(j0);
    for (int i0 = 0; i0 < group; i0 += kHeads) {
      if (i0 > 0) load(j0, i0);
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const float l = i0 + i < group ? lse[i0 + i] : 0.0f;
#pragma unroll
        for (int x = 0; x < kFly; ++x) s[x] += exp2f(z[i][x] - l);
      }
    }
#pragma unroll
    for (int x = 0; x < kFly; ++x)
      if (j0 + x * step < len) c.weights[rec + j0 + x * step] = s[x];
  }
}

__global__ void k_attend_weights(const __grid_constant__ AttendParams p) {
  add_weights(p, blockIdx.z, blockIdx.y, p.lse + static_cast<int64_t>(blockIdx.z) * p.c.num_heads + blockIdx.y * (p.c.num_heads / p.c.num_kv),
              blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x, [] {});
}

// ---------------------------------------------------------------- tiled form
//
// Eight query heads of one key-value head are the rows of a warp's m16n8 MMAs, twice: rows 0-7
// carry the leading part of each head's query (or weights), rows 8-15 the rest of it, so that one
// MMA with the key rows as its B operand gives both partial products and their sum is two
// registers of the same thread. Parts by type of the pages:
//   f16, E4M3 (exact in f16)  two f16 parts, 22 bits, of the query scaled by a power of two and of
//                             the weights scaled by 2^15 (f16's subnormals then lie below 2^-39)
//   bf16                      three bf16 parts, 24 bits: the third in a second MMA
//   f32                       two tf32 parts of both operands, 22 bits
// The register-path MMA is used, not tcgen05: at HBM speed the warp MMAs of a 16-key tile take about a
// third of its time, and their results are where the softmax needs them. The price of eight query
// heads as the rows of a tile is the second reading of the rows by a head group's next block: 16 query
// heads a key-value head (32 x 4096 slots, bf16) 172 to 177 us, 47 % of a copy, for 100 to 107 at
// eight. Keys as the rows, with heads' parts as the columns, would serve more heads from one reading.
//
// Work is cut into tiles of 16 or 32 keys per warp; the tiles of all (sequence, key-value head) units
// are cut into equal runs, so that ragged lengths balance. A block takes a run; where a key-value
// head has more than eight query heads, neighbouring blocks take the same run with eight each, so
// that the second reads the rows from L2. A unit that lies within one run is finished there;
// otherwise each run leaves its partial (o, m, l) and a second kernel joins them in run order.
// Small caches (attend_plan says when) instead give each unit a cluster of blocks with equal shares
// of its tiles, which join through distributed shared memory: one launch. (Joined by the last block
// to arrive, behind a counter, one sequence of 131072 slots took 53 us, the registers of that code
// among it; with the second kernel one key-value head's 131072 slots take 26 us.)

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// 16 bytes, or zeros where `bytes` is 0.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory"); }

__device__ __forceinline__ void mma(__half, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(__nv_bfloat16, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma0(__half, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma0(__nv_bfloat16, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma0(float, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// x = part 0 + part 1 in tf32 (22 bits); the MMA reads the upper 19 bits of part 1.
__device__ __forceinline__ void tf32_parts(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(x - __uint_as_float(hi));
}

// Two values as packed parts of the MMA type.
__device__ __forceinline__ void parts2(float x, float y, uint32_t (&part)[2]) {  // f16
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  part[0] = *reinterpret_cast<const uint32_t*>(&h);
  part[1] = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void parts3(float x, float y, uint32_t (&part)[3]) {  // bf16
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    x -= f.x;
    y -= f.y;
    part[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}

// kFull: head_dim is DP itself, and everything that goes by it is a constant.
template <typename T, int DP, bool kFull>
struct Tiled {
  static constexpr bool kF32 = std::is_same_v<T, float>;
  static constexpr bool kBF16 = std::is_same_v<T, __nv_bfloat16>;
  static constexpr bool kFP8 = std::is_same_v<T, __nv_fp8_e4m3>;
  using M = std::conditional_t<kFP8, __half, T>;  // MMA operand type
  static constexpr int kRow = DP * static_cast<int>(sizeof(T));  // bytes of a row
  static constexpr bool kSwz = kRow % 128 == 0;                  // with kFull: chunks xored by the key
  // the longest pitch of a row in shared memory
  static constexpr int kPitch = kFull ? (kSwz ? kRow : 16 * (((kRow / 16 + 1) & ~1) + 1)) : (kRow == 64 ? 80 : kRow);
  static constexpr int kWarps = kRow <= 512 ? 4 : 2;
  static constexpr int kSub = kRow <= 128 ? 2 : 1;      // 16-key blocks of a warp's tile
  static constexpr int kStages = kRow <= 256 || kRow > 384 ? 3 : 2;
  static constexpr int kThreads = 32 * kWarps;
  // of an SM (three, 168 registers a thread, were slower wherever they fit: rows of 160 bytes 125 us for
  // 105, of 128 bytes 245 for 157)
  static constexpr int kBlocks = kRow <= 384 && DP <= 128 ? 2 : 1;
  static constexpr int kKeys = 16 * kSub * kWarps;  // keys of a block tile
  static constexpr int kLanes = kRow <= 64 ? 4 : 8;  // lanes that copy a row
  static constexpr int kSets = kBF16 ? 2 : 1;
  static constexpr int kSteps = kF32 ? DP / 8 : (kFP8 ? (DP / 16 + 1) & ~1 : DP / 16);  // MMA steps over a head's dims
  static constexpr float kBias = kF32 || kBF16 ? 0.0f : 15.0f;  // log2 of the weights' scale
  static constexpr int kRing = kStages * kWarps * kSub * 32 * kPitch;
  static constexpr int kSmem = kRing + kSets * kSteps * 512;  // and the query's fragments
};

// Beginning and finishing a unit costs a block about as much as kOver tiles: the list that the
// blocks divide has kOver places before each unit's tiles, so that runs of short units (one tile
// each) get fewer of them. With 1, 2 and 4, us: 64 sequences of 1..8191 slots 54.7, 54.1, 58.4; 16 of
// 100..30000 44.7, 43.1, 43.3; 12 of 500..60000 in E4M3 74.0, 71.6, 72.5; 256 of 1..700 51.0, 54.0,
// 62.2; 40 of 10..4000 with heads of 64 21.3, 21.9, 24.0.
constexpr int kOver = 2;

// A tile's place in that list: `at`, of sequence b, unit u, tile of the unit's nt.
struct Cursor {
  int b, kv, tile, nt, len, lo, first;
  int at;
};

__device__ __forceinline__ void cursor_seq(const AttendParams& p, int keys, Cursor& c) {
  int len = p.c.lens[c.b];
  len = len < 0 ? 0 : (len > p.c.max_slots ? p.c.max_slots : len);
  c.len = len;
  c.lo = p.a.window > 0 && !p.c.positions && len > p.a.window ? len - p.a.window : 0;
  c.first = c.lo / keys;
  c.nt = len > 0 ? (len + keys - 1) / keys - c.first : 1;  // an empty sequence still has its zeros to write
}

__device__ __forceinline__ void cursor_next(const AttendParams& p, int keys, Cursor& c) {
  ++c.at;
  if (++c.tile < c.nt) return;
  c.tile = 0;
  c.at += kOver;
  if (++c.kv < p.c.num_kv) return;
  c.kv = 0;
  if (++c.b < p.c.num_seqs) cursor_seq(p, keys, c);
}

__device__ __forceinline__ float exp2_fast(float x) {  // ex2.approx: 2 ulp, 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Each block of a cluster adds its share of the values over all of them, in rank order. Out of line:
// its registers are not the main loop's.
template <typename G>
__device__ __noinline__ void join_cluster(const AttendParams& p, float* s_o, float* s_bm, float* s_bl, int heads, int D, float* out,
                                          float* lse) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), d4 = D / 4;
  for (int i = rank * G::kThreads + threadIdx.x; i < heads * d4; i += p.cluster * G::kThreads) {
    const int h = i / d4, d = 4 * (i - h * d4);
    float m[kMaxCluster], mm = -INFINITY;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      m[r] = r < p.cluster ? cluster.map_shared_rank(s_bm, r)[h] : -INFINITY;
      mm = fmaxf(mm, m[r]);
    }
    const float ref = mm == -INFINITY ? 0.0f : mm;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float ll = 0.0f;
#pragma unroll
    for (int r0 = 0; r0 < kMaxCluster; r0 += 4) {
      float l[4];
      float4 o[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        l[x] = 0.0f;
        o[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r0 + x < p.cluster) {
          l[x] = cluster.map_shared_rank(s_bl, r0 + x)[h];
          o[x] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(s_o, r0 + x) + h * D + d);
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (l[x] == 0.0f) continue;  // no key allowed there, or no tile
        const float f = exp2f(m[r0 + x] - ref);
        v.x += o[x].x * f;
        v.y += o[x].y * f;
        v.z += o[x].z * f;
        v.w += o[x].w * f;
        ll += l[x] * f;
      }
    }
    const float f = ll == 0.0f ? 0.0f : p.c.v_scale / ll;
    float* to = out + h * D + d;
    to[0] = ll == 0.0f ? 0.0f : v.x * f;
    to[1] = ll == 0.0f ? 0.0f : v.y * f;
    to[2] = ll == 0.0f ? 0.0f : v.z * f;
    to[3] = ll == 0.0f ? 0.0f : v.w * f;
    if (lse && d == 0) lse[h] = ll == 0.0f ? INFINITY : ref - G::kBias + log2f(ll);
  }
}

template <typename T, int DP, bool kFull>
__global__ void __launch_bounds__(Tiled<T, DP, kFull>::kThreads, Tiled<T, DP, kFull>::kBlocks) k_attend_tiled(const __grid_constant__ AttendParams p) {
  using G = Tiled<T, DP, kFull>;
  using M = typename G::M;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_sum[G::kWarps], s_rest[G::kWarps];
  __shared__ int s_b, s_off;
  __shared__ float s_bm[8], s_bl[8];  // the block's maximum and sum per head, for its cluster
  __shared__ float s_m[G::kWarps][8], s_l[G::kWarps][8], s_mult[8];
  __shared__ uint32_t s_ok[G::kWarps][G::kStages];
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  const int D = kFull ? DP : c.head_dim;
  const int row_bytes = D * static_cast<int>(sizeof(T)), chunks = row_bytes / 16;
  // Rows of a multiple of 128 bytes (and rows whose pitch would not fit) are stored with their
  // 16-byte chunks xored by the key; others with a pitch of an odd number of chunks. Both keep
  // ldmatrix free of bank conflicts.
  const int pad_chunks = (chunks + 1) & ~1;  // the MMAs read whole steps of 32 bytes
  const bool swz = kFull ? G::kSwz : (row_bytes & 127) == 0 || 16 * (pad_chunks + 1) > G::kPitch;
  const int pitch = swz ? (row_bytes + 127) & ~127 : 16 * (pad_chunks + 1);
  // offset of chunk ch + x of row r, x a constant of a loop whose bits ch leaves clear
  auto chunk_at = [&](int r, int ch, int x) -> uint32_t {
    if constexpr (kFull && G::kSwz) return (r * pitch + ((ch ^ (r & 7)) << 4) ^ ((x & 7) << 4)) + (x >> 3) * 128;
    else return r * pitch + ((swz ? (ch + x) ^ (r & 7) : ch + x) << 4);
  };
  uint8_t* const ring = smem + w * (G::kStages * G::kSub * 32 * pitch);
  const uint32_t ring_addr = pipe::smem_u32(ring);
  uint4* const sq = reinterpret_cast<uint4*>(smem + G::kRing);

  asm volatile("griddepcontrol.launch_dependents;");
  if (pad_chunks != chunks) {  // columns that no copy writes
    for (int i = lane; i < G::kStages * G::kSub * 32; i += 32)
      *reinterpret_cast<uint4*>(ring + i * pitch + ((swz ? chunks ^ (i & 7) : chunks) << 4)) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // This block's run of the list: all units' places, then the sequence that the run begins in.
  // With no more sequences than threads both come from one reading of the lengths.
  auto places = [&](int b) {
    if (b >= c.num_seqs) return 0;
    Cursor s;
    s.b = b;
    cursor_seq(p, G::kKeys, s);
    return (s.nt + kOver) * c.num_kv;
  };
  Cursor cur;
  int t0, t1, n_runs = 1, run = 0, hg, total = 0;
  if (p.cluster > 0) {
    const int unit = blockIdx.x / p.cluster, rank = blockIdx.x - unit * p.cluster;
    hg = unit % p.head_groups;
    cur.b = unit / p.head_groups / c.num_kv;
    cur.kv = unit / p.head_groups - cur.b * c.num_kv;
    cursor_seq(p, G::kKeys, cur);
    t0 = rank * cur.nt / p.cluster;
    t1 = (rank + 1) * cur.nt / p.cluster;
    cur.at = cur.tile = t0;
    if (tid == 0 && (c.lens[cur.b] < 0 || c.lens[cur.b] > c.max_slots)) atomicCAS(c.err, 0, kKvErrSlot);
  } else {
    int mine = places(tid), scan = mine, rest = 0;
    for (int b = tid + G::kThreads; b < c.num_seqs; b += G::kThreads) rest += places(b);
    if (blockIdx.x == 0)
      for (int b = tid; b < c.num_seqs; b += G::kThreads)
        if (c.lens[b] < 0 || c.lens[b] > c.max_slots) atomicCAS(c.err, 0, kKvErrSlot);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
    if (lane == 31) s_sum[w] = scan;
    if (lane == 0) s_rest[w] = rest;
    __syncthreads();
    int before = 0, chunk = 0;
#pragma unroll
    for (int i = 0; i < G::kWarps; ++i) {
      if (i < w) before += s_sum[i];
      chunk += s_sum[i];
      total += s_rest[i];
    }
    total += chunk;
    // A unit cut into P runs costs about P / 50 tiles of joining: runs are at least as long as
    // balances that, and never empty. It shows where few units are long: one key-value head of 50000
    // slots with weights 21.0 us, with the shortest runs 25.8; 30000 slots 13.4 and 13.2. With 1 / 25 and
    // 1 / 200 the batches above take the same times.
    const float tiles = static_cast<float>(total) / static_cast<float>(c.num_seqs * c.num_kv);
    const int shortest = max(1, static_cast<int>(sqrtf(tiles * (1.0f / 50.0f))));
    n_runs = max(1, min(static_cast<int>(gridDim.x) / p.head_groups, total / shortest));
    run = blockIdx.x / p.head_groups;
    hg = blockIdx.x - run * p.head_groups;
    if (run >= n_runs) return;
    t0 = static_cast<int>(static_cast<int64_t>(run) * total / n_runs);
    t1 = static_cast<int>(static_cast<int64_t>(run + 1) * total / n_runs);
    for (int base = 0, acc = 0;;) {
      const int end = acc + before + scan;  // of this thread's sequence
      if (end - mine <= t0 && t0 < end) {
        s_b = base + tid;
        s_off = t0 - (end - mine);
      }
      acc += chunk;
      if (t0 < acc) break;
      base += G::kThreads;
      mine = scan = places(base + tid);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += y;
      }
      __syncthreads();
      if (lane == 31) s_sum[w] = scan;
      __syncthreads();
      before = chunk = 0;
#pragma unroll
      for (int i = 0; i < G::kWarps; ++i) {
        if (i < w) before += s_sum[i];
        chunk += s_sum[i];
      }
    }
    __syncthreads();
    cur.b = s_b;
    cursor_seq(p, G::kKeys, cur);
    cur.kv = s_off / (cur.nt + kOver);
    cur.tile = s_off - cur.kv * (cur.nt + kOver) - kOver;
    cur.at = t0;
    if (cur.tile < 0) {
      cur.at -= cur.tile;
      cur.tile = 0;
    }
  }
  Cursor nxt = cur;
  const int cur_b = cur.b, cur_kv = cur.kv;  // a cluster's unit

  // Copies the warp's keys and values of the tile at `nxt`; rows that the mask leaves out are
  // zeros (their contents, even NaN, must not reach the sums).
  const bool one_page = c.page_size % 16 == 0 && !(p.a.window > 0 && c.positions);
  constexpr int kRows = 32 / G::kLanes;  // rows copied at a time
  const int lr = lane / G::kLanes, lc = lane % G::kLanes;
  auto page_of = [&](int j, int& in) {
    const int slot_page = p.page_shift >= 0 ? j >> p.page_shift : j / c.page_size;
    in = j - slot_page * c.page_size;
    return c.table[nxt.b * c.table_stride + slot_page];
  };
  auto offset = [](const KvBytes& s, int page, int in, int kv) {  // 32 x 32 -> 64 bit products
    return static_cast<uint64_t>(static_cast<uint32_t>(page)) * s.page + static_cast<uint64_t>(static_cast<uint32_t>(in)) * s.slot +
           static_cast<uint64_t>(static_cast<uint32_t>(kv)) * s.head;
  };
  auto issue = [&](int stage) {
    if (nxt.at < t1) {
      uint32_t ok_all = 0;
#pragma unroll
      for (int sb = 0; sb < G::kSub; ++sb) {
        const int j0 = (nxt.first + nxt.tile) * G::kKeys + 16 * (G::kSub * w + sb);
        const uint32_t dst = ring_addr + (stage * G::kSub + sb) * 32 * pitch;
        uint32_t okm;
        if (one_page) {
          // the 16 slots lie in one page, and their rows a stride apart
          const int from = min(max(nxt.lo - j0, 0), 16), to = min(max(nxt.len - j0, 0), 16);
          okm = ((1u << to) - 1u) & ~((1u << from) - 1u);
          int page = 0, in = 0;
          if (okm != 0) {
            page = page_of(j0, in);
            if (page < 0 || page >= c.num_pages) {
              if (lane == 0) atomicCAS(c.err, 0, kKvErrPage);
              page = in = 0;
              okm = 0;
            }
          }
          const uint64_t ko = offset(p.kb, page, in + lr, nxt.kv);
          const uint8_t* ks = c.k.base + ko + 16 * lc;
          const uint8_t* vs = c.v.base + (p.same ? ko : offset(p.vb, page, in + lr, nxt.kv)) + 16 * lc;
#pragma unroll
          for (int r0 = 0; r0 < 16; r0 += kRows) {
            const int n = (okm >> (r0 + lr)) & 1 ? 16 : 0;
#pragma unroll
            for (int x = 0; x < G::kRow / 16; x += G::kLanes) {
              if (((kFull && G::kRow / 16 - x >= G::kLanes)) || x + lc < chunks) {
                uint32_t at;
                if constexpr (kFull && G::kSwz) at = (r0 + lr) * pitch + (((lc ^ lr) ^ (r0 & 7)) << 4) + 16 * x;
                else at = (r0 + lr) * pitch + ((swz ? (x + lc) ^ ((r0 + lr) & 7) : x + lc) << 4);
                cp16(dst + at, ks + 16 * x, n);
                cp16(dst + 16 * pitch + at, vs + 16 * x, n);
              }
            }
            ks += static_cast<uint64_t>(p.kb.slot) * kRows;
            vs += static_cast<uint64_t>(p.vb.slot) * kRows;
          }
        } else {
          const int j = j0 + (lane & 15);
          bool ok = j >= nxt.lo && j < nxt.len;
          uint64_t ko = 0, vo = 0;
          if (ok) {
            int in;
            const int page = page_of(j, in);
            if (p.a.window > 0 && c.positions) {
              const int64_t rec = (static_cast<int64_t>(nxt.b) * c.num_kv + nxt.kv) * c.max_slots + j;
              ok = c.positions[rec] > c.seen[nxt.b] - 1 - p.a.window;
            }
            if (page < 0 || page >= c.num_pages) {
              atomicCAS(c.err, 0, kKvErrPage);
              ok = false;
            }
            if (ok) {
              ko = offset(p.kb, page, in, nxt.kv);
              vo = p.same ? ko : offset(p.vb, page, in, nxt.kv);
            }
          }
          okm = __ballot_sync(0xffffffffu, ok) & 0xffffu;
#pragma unroll
          for (int r0 = 0; r0 < 16; r0 += kRows) {
            const int r = r0 + lr;
            const uint64_t kr = __shfl_sync(0xffffffffu, ko, r), vr = p.same ? kr : __shfl_sync(0xffffffffu, vo, r);
            const int n = (okm >> r) & 1 ? 16 : 0;
#pragma unroll
            for (int x = 0; x < G::kRow / 16; x += G::kLanes) {
              if (x + lc < chunks) {
                const uint32_t at = r * pitch + ((swz ? (x + lc) ^ (r & 7) : x + lc) << 4);
                cp16(dst + at, c.k.base + kr + 16 * (x + lc), n);
                cp16(dst + 16 * pitch + at, c.v.base + vr + 16 * (x + lc), n);
              }
            }
          }
        }
        ok_all |= okm << (16 * sb);
      }
      if (lane == 0) s_ok[w][stage] = ok_all;
      cursor_next(p, G::kKeys, nxt);
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < G::kStages - 1; ++s) issue(s);

  float o[DP / 8][2];
  float m = -INFINITY, l = 0.0f, mult = 0.0f, slope = 0.0f;
  int stage = 0, q_pos = 0;
  bool fresh = true;  // the unit's query is not in shared memory yet
  int unit_start = 0;

  while (cur.at < t1) {
    __syncwarp();  // the slot of the tile before has been read by every lane
    issue(stage == 0 ? G::kStages - 1 : stage - 1);
    const int kv = cur.kv, h0 = 8 * hg;
    const int heads = p.group - h0 < 8 ? p.group - h0 : 8;  // of this unit
    const int head = kv * p.group + h0;                      // the first of them
    if (fresh) {
      fresh = false;
      unit_start = cur.at - cur.tile;  // place of the unit's first tile
      q_pos = c.positions ? c.seen[cur.b] - 1 : cur.len - 1;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[i][e] = 0.0f;
      m = -INFINITY;
      l = 0.0f;
      const float* q = p.a.q + cur.b * p.a.q_ld + static_cast<int64_t>(head) * D;
      const float base = p.a.scale * c.k_scale * kLog2e;
      // kPer threads a head, each with its share of the head's fragments
      constexpr int kPer = G::kThreads / 8, kVals = G::kF32 ? 2 : 4, kEnt = (G::kSteps * 4 + kPer - 1) / kPer;
      const int h = tid / kPer;
      float v[kEnt][kVals];
      float mx = 0.0f;
#pragma unroll
      for (int x = 0; x < kEnt; ++x) {
        const int i = tid % kPer + x * kPer, step = i >> 2, tt = i & 3;
#pragma unroll
        for (int y = 0; y < kVals; ++y) {
          const int d = G::kF32 ? 8 * step + tt + 4 * y : 16 * step + (G::kFP8 ? 4 * tt + y : 2 * tt + (y & 1) + 8 * (y >> 1));
          v[x][y] = h < heads && d < D ? q[h * D + d] : 0.0f;
          mx = fmaxf(mx, fabsf(v[x][y]));
        }
      }
      float f = 1.0f;
      if constexpr (!G::kF32 && !G::kBF16) {
        // a power of two that brings the head's largest |q| to [2^13, 2^14)
#pragma unroll
        for (int x = kPer / 2; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        if (mx > 0.0f && mx < INFINITY) f = ldexpf(1.0f, min(126, 13 - ilogbf(mx)));
        if (tid % kPer == 0) s_mult[h] = f;
      }
#pragma unroll
      for (int x = 0; x < kEnt; ++x) {
        const int i = tid % kPer + x * kPer;
        if (i >= G::kSteps * 4) break;
        const int at = (i >> 2) * 32 + 4 * h + (i & 3);
        if constexpr (G::kF32) {
          uint32_t a[4];
          tf32_parts(v[x][0], a[0], a[1]);
          tf32_parts(v[x][1], a[2], a[3]);
          sq[at] = make_uint4(a[0], a[1], a[2], a[3]);
        } else if constexpr (G::kBF16) {
          uint32_t lo[3], hi[3];
          parts3(v[x][0], v[x][1], lo);
          parts3(v[x][2], v[x][3], hi);
          sq[at] = make_uint4(lo[0], lo[1], hi[0], hi[1]);
          sq[G::kSteps * 32 + at] = make_uint4(lo[2], 0u, hi[2], 0u);
        } else {
          uint32_t lo[2], hi[2];
          parts2(v[x][0] * f, v[x][1] * f, lo);
          parts2(v[x][2] * f, v[x][3] * f, hi);
          sq[at] = make_uint4(lo[0], lo[1], hi[0], hi[1]);
        }
      }
      __syncthreads();
      mult = G::kF32 || G::kBF16 ? base : base / s_mult[g];
      slope = p.a.alibi ? alibi_slope(head + g, c.num_heads) * kLog2e : 0.0f;
    }

    cp_wait<G::kStages - 1>();
    __syncwarp();
    const uint32_t kbase = ring_addr + stage * G::kSub * 32 * pitch, vbase = kbase + 16 * pitch;
    const uint32_t okm = s_ok[w][stage];
    const int j0 = (cur.first + cur.tile) * G::kKeys + 16 * G::kSub * w;
    constexpr int kN = 2 * G::kSub;  // blocks of eight keys
    constexpr int kFold = G::kF32 ? 16 : (std::is_same_v<T, __half> ? 32 : 64);  // dims

    // Scores of keys j0 + 8 n + 2 t + e for head g. The MMAs cut their sums short of the last bit, so
    // that a chain over all of a row leans towards zero: kFold dims' products start from zero, and both
    // parts of the query are added to the score in rounded fp32. Error of the result against 64 bits,
    // chained and so, with the formula in fp32 (one running sum a score) for comparison: f32 rows of
    // 256, 1.6e-6, 2.9e-7 and 7.0e-7; bf16 of 256, 1.1e-6, 3.5e-7 and 5.8e-7; one short bf16 sequence,
    // 6.5e-7, 3.7e-7 and 6.8e-7; at the times of the chain within 1 % (32 dims in bf16 as well: 2.9e-7
    // on the short one, and 1.6 % longer on a ragged batch).
    float z[kN][2];
    float s[kN][4];
    auto fold = [&](bool first) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) z[n][e] = first ? s[n][e] + s[n][e + 2] : z[n][e] + (s[n][e] + s[n][e + 2]);
    };
    if constexpr (G::kF32) {
#pragma unroll
      for (int st = 0; st < G::kSteps; st += 2) {
        if (8 * st < D) {
          const bool begins = 8 * st % kFold == 0;
          uint32_t a0[4], a1[4];
          *reinterpret_cast<uint4*>(a0) = sq[st * 32 + lane];
          *reinterpret_cast<uint4*>(a1) = sq[(st + 1) * 32 + lane];
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            // four chunks (16 dims) of eight keys
            uint32_t k[4], hi[4], lo[4];
            ldsm4(k, kbase + (n >> 1) * 32 * pitch + chunk_at(8 * (n & 1) + (lane & 7), lane >> 3, 2 * st));
#pragma unroll
            for (int e = 0; e < 4; ++e) tf32_parts(__uint_as_float(k[e]), hi[e], lo[e]);
            if (begins) mma0(M(), s[n], a0, lo[0], lo[1]);
            else mma(M(), s[n], a0, lo[0], lo[1]);
            mma(M(), s[n], a0, hi[0], hi[1]);
            if (8 * st + 8 < D) {
              mma(M(), s[n], a1, lo[2], lo[3]);
              mma(M(), s[n], a1, hi[2], hi[3]);
            }
          }
          if ((8 * st + 16) % kFold == 0 || 8 * st + 16 >= D) fold(8 * st < kFold);
        }
      }
    } else if constexpr (G::kFP8) {
#pragma unroll
      for (int st = 0; st < G::kSteps; st += 2) {
        if (16 * st < D) {
          const bool begins = 16 * st % kFold == 0;
          uint32_t k[G::kSub][4];
#pragma unroll
          for (int sb = 0; sb < G::kSub; ++sb)
            ldsm4(k[sb], kbase + sb * 32 * pitch + chunk_at(8 * ((lane >> 3) & 1) + (lane & 7), lane >> 4, st));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t a[4];
            *reinterpret_cast<uint4*>(a) = sq[(st + x) * 32 + lane];
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              uint32_t b0, b1;
              e4m3_pairs(k[n >> 1][2 * x + (n & 1)], b0, b1);
              if (begins && x == 0) mma0(M(), s[n], a, b0, b1);
              else mma(M(), s[n], a, b0, b1);
            }
          }
          if ((16 * st + 32) % kFold == 0 || 16 * st + 32 >= D) fold(16 * st < kFold);
        }
      }
    } else {
#pragma unroll
      for (int st = 0; st < G::kSteps; ++st) {
        if (16 * st < D) {
          const bool begins = 16 * st % kFold == 0;
          uint32_t k[G::kSub][4];
#pragma unroll
          for (int sb = 0; sb < G::kSub; ++sb)
            ldsm4(k[sb], kbase + sb * 32 * pitch + chunk_at(8 * (lane >> 4) + (lane & 7), (lane >> 3) & 1, 2 * st));
#pragma unroll
          for (int x = 0; x < G::kSets; ++x) {
            uint32_t a[4];
            *reinterpret_cast<uint4*>(a) = sq[(x * G::kSteps + st) * 32 + lane];
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              const uint32_t b0 = k[n >> 1][2 * (n & 1)], b1 = k[n >> 1][2 * (n & 1) + 1];
              if (begins && x == 0) mma0(M(), s[n], a, b0, b1);
              else mma(M(), s[n], a, b0, b1);
            }
          }
          if ((16 * st + 16) % kFold == 0 || 16 * st + 16 >= D) fold(16 * st < kFold);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) z[n][e] *= mult;
    if (p.a.alibi) {
      const int32_t* pos = c.positions ? c.positions + (static_cast<int64_t>(cur.b) * c.num_kv + kv) * c.max_slots : nullptr;
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 8 * n + 2 * t + e;
          if ((okm >> i) & 1) z[n][e] -= slope * static_cast<float>(q_pos - (pos ? pos[j0 + i] : j0 + i));
        }
    }
    if (okm != (G::kSub == 2 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (!((okm >> (8 * n + 2 * t + e)) & 1)) z[n][e] = -INFINITY;
    }
    if (p.a.accumulate && g < heads) {
      float* sc = p.scores + (static_cast<int64_t>(cur.b) * c.num_heads + head + g) * c.max_slots + j0;
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (j0 + 8 * n + 2 * t + e < cur.len) sc[8 * n + 2 * t + e] = z[n][e];
    }
    float mx = fmaxf(z[0][0], z[0][1]);
#pragma unroll
    for (int n = 1; n < kN; ++n) mx = fmaxf(mx, fmaxf(z[n][0], z[n][1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (__any_sync(0xffffffffu, mx > m)) {
      const float m_new = fmaxf(m, mx);
      const float corr = m == -INFINITY ? 0.0f : exp2_fast(m - m_new);
      l *= corr;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[i][e] *= corr;
      m = m_new;
    }
    const float ref = (m == -INFINITY ? 0.0f : m) - G::kBias;
    float pw[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pw[n][e] = exp2_fast(z[n][e] - ref);
        l += pw[n][e];
      }

    // o += weights . values. The MMAs' accumulators cut their sums short of the last bit: a tile's
    // sum starts from zero and is added to o (both parts of the weights at once) in rounded fp32, or
    // runs of hundreds of tiles would lose a digit (E4M3, 30k..131k slots: 3.3e-6 of the result).
    if constexpr (G::kF32) {
      uint32_t a[kN][4];  // k index t is key 2 t, t + 4 is key 2 t + 1
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        tf32_parts(pw[n][0], a[n][0], a[n][1]);
        tf32_parts(pw[n][1], a[n][2], a[n][3]);
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        if (8 * i < D) {
          float d[4];
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            const int r0 = 8 * (n & 1) + 2 * t, r1 = r0 + 1;
            const uint32_t vb = vbase + (n >> 1) * 32 * pitch;
            const float v0 = __uint_as_float(lds32(vb + chunk_at(r0, g >> 2, 2 * i) + 4 * (g & 3)));
            const float v1 = __uint_as_float(lds32(vb + chunk_at(r1, g >> 2, 2 * i) + 4 * (g & 3)));
            uint32_t h0, l0, h1, l1;
            tf32_parts(v0, h0, l0);
            tf32_parts(v1, h1, l1);
            if (n == 0) mma0(M(), d, a[n], l0, l1);
            else mma(M(), d, a[n], l0, l1);
            mma(M(), d, a[n], h0, h1);
          }
          o[i][0] += d[0] + d[2];
          o[i][1] += d[1] + d[3];
        }
      }
    } else {
      uint32_t a[G::kSub][G::kSets][4];
#pragma unroll
      for (int sb = 0; sb < G::kSub; ++sb) {
        const float(&p0)[2] = pw[2 * sb], (&p1)[2] = pw[2 * sb + 1];
        if constexpr (G::kBF16) {
          uint32_t x[3], y[3];
          parts3(p0[0], p0[1], x);
          parts3(p1[0], p1[1], y);
          a[sb][0][0] = x[0]; a[sb][0][1] = x[1]; a[sb][0][2] = y[0]; a[sb][0][3] = y[1];
          a[sb][1][0] = x[2]; a[sb][1][1] = 0u; a[sb][1][2] = y[2]; a[sb][1][3] = 0u;
        } else {
          uint32_t x[2], y[2];
          parts2(p0[0], p0[1], x);
          parts2(p1[0], p1[1], y);
          a[sb][0][0] = x[0]; a[sb][0][1] = x[1]; a[sb][0][2] = y[0]; a[sb][0][3] = y[1];
        }
      }
      const int r = 8 * ((lane >> 3) & 1) + (lane & 7);
      constexpr int kWide = G::kFP8 ? 4 : 2;  // n8 tiles of an ldmatrix
#pragma unroll
      for (int i = 0; i < DP / 8; i += kWide) {
        if (8 * i < D) {
          float d[kWide][4];
#pragma unroll
          for (int sb = 0; sb < G::kSub; ++sb) {
            uint32_t v[4];
            ldsm4t(v, vbase + sb * 32 * pitch + chunk_at(r, lane >> 4, G::kFP8 ? i / 2 : i));
            auto add = [&](int x, const uint32_t(&w)[4], uint32_t b0, uint32_t b1, bool first) {
              if (first) mma0(M(), d[x], w, b0, b1);
              else mma(M(), d[x], w, b0, b1);
            };
            if constexpr (G::kFP8) {
              // a register holds dims 2 g, 2 g + 1 of keys 2 t, 2 t + 1: regroup the bytes by dim
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                if (i + 2 * x >= DP / 8) break;
                uint32_t e0, o0, e1, o1;
                e4m3_pairs(__byte_perm(v[2 * x], 0, 0x3120), e0, o0);
                e4m3_pairs(__byte_perm(v[2 * x + 1], 0, 0x3120), e1, o1);
                add(2 * x, a[sb][0], e0, e1, sb == 0);
                add(2 * x + 1, a[sb][0], o0, o1, sb == 0);
              }
            } else {
#pragma unroll
              for (int x = 0; x < G::kSets; ++x) {  // the least part first
                const int set = G::kSets - 1 - x;
                add(0, a[sb][set], v[0], v[1], sb == 0 && x == 0);
                add(1, a[sb][set], v[2], v[3], sb == 0 && x == 0);
              }
            }
          }
#pragma unroll
          for (int x = 0; x < kWide; ++x) {
            if (i + x >= DP / 8) break;
            o[i + x][0] += d[x][0] + d[x][2];
            o[i + x][1] += d[x][1] + d[x][3];
          }
        }
      }
    }
    const bool unit_ends = cur.tile + 1 == cur.nt;
    if (unit_ends || cur.at + 1 == t1) {
      // Join the warps: each leaves its sums in the slot it has just read (rows of D values, turned by
      // four per head against bank conflicts), then every thread adds the four of its values.
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) {
        s_m[w][g] = m;
        s_l[w][g] = l;
      }
      uint8_t* const scratch = ring + stage * G::kSub * 32 * pitch;
      float* const mine = reinterpret_cast<float*>(scratch) + g * D;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < DP / 8; i += G::kFP8 ? 2 : 1) {
        if (8 * i >= D) break;
        int d = (G::kFP8 ? 8 * i + 4 * t : 8 * i + 2 * t) + 4 * g;
        if (d >= D) d -= D;
        const float2 a = make_float2(o[i][0], o[i][1]);
        if constexpr (G::kFP8) {
          *reinterpret_cast<float4*>(mine + d) = make_float4(a.x, o[i + 1][0], a.y, o[i + 1][1]);
        } else {
          *reinterpret_cast<float2*>(mine + d) = a;
        }
      }
      __syncthreads();
      const bool whole = unit_ends && unit_start >= t0;
      float* out = p.a.out + cur.b * p.a.out_ld + static_cast<int64_t>(head) * D;
      // a run leaves at most two partial units: one that began before it, one that goes on after it
      const int stride = D + 4;  // 16-byte rows
      float* dst = p.part + (2ll * blockIdx.x + (unit_start >= t0 ? 1 : 0)) * 8 * stride;
      const int d4 = D / 4;
      for (int i = tid; i < heads * d4; i += G::kThreads) {
        const int h = i / d4, d = 4 * (i - h * d4);
        float mm = s_m[0][h];
#pragma unroll
        for (int x = 1; x < G::kWarps; ++x) mm = fmaxf(mm, s_m[x][h]);
        const float r = mm == -INFINITY ? 0.0f : mm;
        int at = d + 4 * h;
        if (at >= D) at -= D;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float ll = 0.0f;
#pragma unroll
        for (int x = 0; x < G::kWarps; ++x) {
          const float f = exp2f(s_m[x][h] - r);
          const float4 y = *reinterpret_cast<const float4*>(smem + (x * G::kStages + stage) * (G::kSub * 32 * pitch) + (h * D + at) * 4);
          v.x += y.x * f;
          v.y += y.y * f;
          v.z += y.z * f;
          v.w += y.w * f;
          ll += s_l[x][h] * f;
        }
        if (p.cluster > 0) {
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(sq) + h * D + d) = v;
          if (d == 0) {
            s_bm[h] = mm;
            s_bl[h] = ll;
          }
        } else if (whole) {
          const float f = ll == 0.0f ? 0.0f : c.v_scale / ll;
          float* to = out + h * D + d;
          to[0] = ll == 0.0f ? 0.0f : v.x * f;
          to[1] = ll == 0.0f ? 0.0f : v.y * f;
          to[2] = ll == 0.0f ? 0.0f : v.z * f;
          to[3] = ll == 0.0f ? 0.0f : v.w * f;
          if (p.a.accumulate && d == 0)
            p.lse[static_cast<int64_t>(cur.b) * c.num_heads + head + h] = ll == 0.0f ? INFINITY : r - G::kBias + log2f(ll);
        } else {
          *reinterpret_cast<float4*>(dst + h * stride + d) = v;
          if (d == 0) {
            dst[h * stride + D] = mm;
            dst[h * stride + D + 1] = ll;
          }
        }
      }
      if (p.cluster == 0 && unit_start >= t0 && hg == 0 && tid == 0) {  // the run that began the unit says where its parts are
        const int last = static_cast<int>((static_cast<int64_t>(unit_start + cur.nt) * n_runs - 1) / total);
        p.spans[cur.b * c.num_kv + kv] = make_int2(run, last - run + 1);
      }
      __syncthreads();  // the slots are copies' again, and the next unit's query may come
      if (pad_chunks != chunks) {
        for (int i = lane; i < G::kSub * 32; i += 32)
          *reinterpret_cast<uint4*>(scratch + i * pitch + ((swz ? chunks ^ (i & 7) : chunks) << 4)) = make_uint4(0, 0, 0, 0);
      }
      fresh = true;
    }
    stage = stage + 1 == G::kStages ? 0 : stage + 1;
    cursor_next(p, G::kKeys, cur);
  }
  cp_wait<0>();
  if (p.cluster == 0) return;

  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int heads = min(p.group - 8 * hg, 8), head = cur_kv * p.group + 8 * hg, rank = static_cast<int>(cluster.block_rank());
  if (t0 == t1 && tid < 8) {  // a block without tiles has nothing to add
    s_bm[tid] = -INFINITY;
    s_bl[tid] = 0.0f;
  }
  cluster.sync();
  join_cluster<G>(p, reinterpret_cast<float*>(sq), s_bm, s_bl, heads, D,
                  p.a.out + cur_b * p.a.out_ld + static_cast<int64_t>(head) * D,
                  p.a.accumulate ? p.lse + static_cast<int64_t>(cur_b) * c.num_heads + head : nullptr);
  if (p.a.accumulate && rank == 0 && hg == 0 && tid == 0) p.spans[cur_b * c.num_kv + cur_kv] = make_int2(0, 1);
  cluster.sync();  // no block leaves while another reads its shared memory
}

// What is left once all runs are done. Blocks below num_heads join the parts of one query head in
// order (the unit's first run left its second slot, the others their first; the warps take the parts
// in turn, each with its running maximum; their sums are added in warp order). The others, with
// accumulate, add the attention weights of a key-value head's slots; the normalisers of split units
// they make for themselves. Latency bound: four warps a block and registers for nine blocks an SM, so
// that many short joins run at once (64 sequences of 32 heads, ragged: 54.4 us with the attention, 55.4
// with seven an SM), or sixteen warps where units have many parts (one key-value head of 131072
// slots, 296 parts: 26.3 us for 41.8; 56 heads of 8191, 5 parts each, with weights: 53.1 for 54.7).
constexpr int kMaxGroup = 128;  // query heads of a key-value head that the weights' blocks can hold
constexpr int kManyParts = 4;   // parts of a unit, on average, beyond which sixteen warps join them

template <int kBias, bool kWide, int kW>  // kWide: head_dim > 128
__global__ void __launch_bounds__(32 * kW, kW == 4 ? 9 : 2) k_attend_finish(const __grid_constant__ AttendParams p) {
  __shared__ float s_o[kW][kWide ? 256 : 128];
  __shared__ float s_m[kW], s_l[kW];
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const KvView& c = p.c;
  const int b = blockIdx.y, D = c.head_dim, stride = D + 4;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  // row of part i of query head r of a key-value head
  auto part_of = [&](int first_run, int r, int i) {
    return p.part + ((static_cast<int64_t>(first_run + i) * p.head_groups + (r >> 3)) * 2 + (i == 0)) * 8 * stride + (r & 7) * stride;
  };
  if (static_cast<int>(blockIdx.x) >= c.num_heads) {
    const int at = blockIdx.x - c.num_heads, kv = at % c.num_kv, chunk = at / c.num_kv, chunks = (gridDim.x - c.num_heads) / c.num_kv;
    float* lse = &s_o[0][0];
    add_weights(p, b, kv, lse, chunk * (32 * kW) + threadIdx.x, chunks * (32 * kW), [&] {
      const int2 span = p.spans[static_cast<int64_t>(b) * c.num_kv + kv];
      for (int r = w; r < p.group; r += kW) {
        if (span.y <= 1) {
          if (lane == 0) lse[r] = p.lse[static_cast<int64_t>(b) * c.num_heads + kv * p.group + r];
          continue;
        }
        float m = -INFINITY, l = 0.0f;
        for (int i = lane; i < span.y; i += 32) {  // a lane's parts, then the lanes'
          const float* part = part_of(span.x, r, i) + D;
          const float pm = __ldcg(part), pl = __ldcg(part + 1), both = fmaxf(m, pm), ref = both == -INFINITY ? 0.0f : both;
          l = l * exp2f(m - ref) + pl * exp2f(pm - ref);
          m = both;
        }
        float all = m;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, x));
        const float ref = all == -INFINITY ? 0.0f : all;
        l = warp_sum(l * exp2f(m - ref));
        if (lane == 0) lse[r] = l == 0.0f ? INFINITY : ref - kBias + log2f(l);
      }
      __syncthreads();
    });
    return;
  }
  const int h = blockIdx.x, kv = h / p.group, r = h - kv * p.group;
  const int2 span = p.spans[static_cast<int64_t>(b) * c.num_kv + kv];
  if (span.y <= 1) return;
  constexpr int kRows = kWide ? 2 : 1, kBatch = 4 / kRows;  // float4s of a lane, parts in flight
  float4 v[kRows] = {};
  float m = -INFINITY, l = 0.0f;
  for (int i0 = w; i0 < span.y; i0 += kW * kBatch) {
    float4 row[kBatch][kRows];
    float ms[kBatch], ls[kBatch];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int i = i0 + kW * x;
      ms[x] = -INFINITY;
      ls[x] = 0.0f;
#pragma unroll
      for (int e = 0; e < kRows; ++e) row[x][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i < span.y) {
        const float* src = part_of(span.x, r, i);
        ms[x] = __ldcg(src + D);
        ls[x] = __ldcg(src + D + 1);
#pragma unroll
        for (int e = 0; e < kRows; ++e)
          if (4 * lane + 128 * e < D) row[x][e] = __ldcg(reinterpret_cast<const float4*>(src + 4 * lane + 128 * e));
      }
    }
    float m_new = m;
#pragma unroll
    for (int x = 0; x < kBatch; ++x) m_new = fmaxf(m_new, ms[x]);
    const float ref = m_new == -INFINITY ? 0.0f : m_new, f = exp2_fast(m - ref);
    l *= f;
#pragma unroll
    for (int e = 0; e < kRows; ++e) v[e] = make_float4(v[e].x * f, v[e].y * f, v[e].z * f, v[e].w * f);
    m = m_new;
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const float fx = exp2_fast(ms[x] - ref);
      l += ls[x] * fx;
#pragma unroll
      for (int e = 0; e < kRows; ++e) {
        v[e].x += row[x][e].x * fx;
        v[e].y += row[x][e].y * fx;
        v[e].z += row[x][e].z * fx;
        v[e].w += row[x][e].w * fx;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kRows; ++e)
    if (4 * lane + 128 * e < D) *reinterpret_cast<float4*>(&s_o[w][4 * lane + 128 * e]) = v[e];
  if (lane == 0) {
    s_m[w] = m;
    s_l[w] = l;
  }
  __syncthreads();
  m = s_m[0];
#pragma unroll
  for (int x = 1; x < kW; ++x) m = fmaxf(m, s_m[x]);
  const float ref = m == -INFINITY ? 0.0f : m;
  float* out = p.a.out + b * p.a.out_ld + static_cast<int64_t>(h) * D;
  for (int d = threadIdx.x; d < D; d += 32 * kW) {
    float sum = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int x = 0; x < kW; ++x) {
      const float f = exp2_fast(s_m[x] - ref);
      l += s_l[x] * f;
      sum += s_o[x][d] * f;
    }
    out[d] = l == 0.0f ? 0.0f : sum * (c.v_scale / l);
  }
}

int simple_splits(const KvView& v) {
  const int64_t rows = static_cast<int64_t>(v.num_seqs) * v.num_heads;
  int64_t s = (148 * 16 + rows - 1) / rows;
  s = std::min<int64_t>(s, (v.max_slots + 127) / 128);
  s = std::min<int64_t>(s, 64);
  return s < 1 ? 1 : static_cast<int>(s);
}

// The tiled form copies rows in 16-byte pieces and multiplies 32-bit strides and counts.
bool tiled(const KvView& v, KvType type) {
  const int size = kv_size(type);
  for (const KvPool& p : {v.k, v.v})
    for (int64_t s : {p.page, p.slot, p.head})
      if (s * size > 0xffffffffll) return false;
  const int64_t units = static_cast<int64_t>(v.num_seqs) * v.num_kv;
  if (units * (v.max_slots / 32 + 1 + kOver) > 0x7fffffffll) return false;  // a tile has 32 keys or more
  if (v.num_heads / v.num_kv > kMaxGroup) return false;
  return v.head_dim % 8 == 0 && v.head_dim * size % 16 == 0 && pool_aligned(v.k, size, 16) && pool_aligned(v.v, size, 16);
}

template <typename F>
Status by_shape(const KvView& v, KvType type, F&& f) {
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (v.head_dim == 64) return f(Tiled<T, 64, true>{}, k_attend_tiled<T, 64, true>);
    if (v.head_dim == 80) return f(Tiled<T, 80, true>{}, k_attend_tiled<T, 80, true>);
    if (v.head_dim == 96) return f(Tiled<T, 96, true>{}, k_attend_tiled<T, 96, true>);
    if (v.head_dim == 128) return f(Tiled<T, 128, true>{}, k_attend_tiled<T, 128, true>);
    if (v.head_dim == 256) return f(Tiled<T, 256, true>{}, k_attend_tiled<T, 256, true>);
    if (v.head_dim < 64) return f(Tiled<T, 64, false>{}, k_attend_tiled<T, 64, false>);
    if (v.head_dim < 128) return f(Tiled<T, 128, false>{}, k_attend_tiled<T, 128, false>);
    return f(Tiled<T, 256, false>{}, k_attend_tiled<T, 256, false>);
  });
}

int head_groups(const KvView& v) { return (v.num_heads / v.num_kv + 7) / 8; }

} // namespace

Status attend_plan(KvCache* c) {
  const KvView& v = c->view;
  const size_t rows = static_cast<size_t>(v.num_seqs) * v.num_heads;
  c->attend_tiled = tiled(v, c->type);
  if (!c->attend_tiled) {
    c->part_bytes = rows * simple_splits(v) * (v.head_dim + 2) * 4;
    return Status::Ok();
  }
  return by_shape(v, c->type, [&](auto g, auto* kernel) {
    using G = decltype(g);
    WB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem));
    int per_sm = 0, sms = 0;
    WB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, G::kThreads, G::kSmem));
    WB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c->device));
    if (per_sm < 1) return Status::Internal("kv attend: the kernel does not fit");
    const int64_t units = static_cast<int64_t>(v.num_seqs) * v.num_kv;
    const int64_t most = units * ((v.max_slots + G::kKeys - 1) / G::kKeys + kOver);
    const int hg = head_groups(v);
    c->attend_blocks = static_cast<int>(std::min<int64_t>(std::max(1, per_sm * sms / hg), most)) * hg;
    c->part_bytes = static_cast<size_t>(c->attend_blocks) * 2 * 8 * (v.head_dim + 4) * 4;
    // Clusters where all of them are resident together and a block's tiles are so few that ragged
    // lengths cannot cost more than the second launch (one sequence of 500 slots, 16 heads: 6.1 us
    // against 7.3; with 16 tiles a block they are the slower form, 19 us against 17).
    const int64_t tiles = (v.max_slots + G::kKeys - 1) / G::kKeys;
    int size = kMaxCluster;
    while (size > 1 && (units * hg * size > static_cast<int64_t>(per_sm) * sms || size > tiles)) size /= 2;
    if (size > 1 && tiles <= 4 * size) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      cfg.blockDim = dim3(G::kThreads);
      cfg.dynamicSmemBytes = G::kSmem;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      for (int fit = 0; size > 1; size /= 2) {
        at[0].val.clusterDim = {static_cast<unsigned>(size), 1, 1};
        cfg.gridDim = dim3(static_cast<unsigned>(units * hg * size));
        WB_CUDA(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
        if (fit >= units * hg) break;
      }
      if (size > 1 && tiles <= 4 * size) c->attend_cluster = size;
    }
    c->span_bytes = static_cast<size_t>(units) * 8;
    return Status::Ok();
  });
}

Status kv_attend(KvCache* c, const KvAttendArgs& a, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(c->device));
  AttendParams p;
  p.a = a;
  p.c = c->view;
  const KvView& v = c->view;
  if (a.lens) p.c.lens = const_cast<int32_t*>(a.lens);  // read only
  if (!(p.a.scale > 0.0f)) p.a.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(v.head_dim)));
  if (!p.a.weights_in) p.a.weights_in = v.weights;
  p.part = c->part;
  p.scores = c->scores;
  p.lse = c->lse;
  p.group = v.num_heads / v.num_kv;
  p.head_groups = head_groups(v);
  p.page_shift = (v.page_size & (v.page_size - 1)) == 0 ? 31 - __builtin_clz(v.page_size) : -1;
  p.spans = reinterpret_cast<int2*>(c->spans);
  const unsigned B = v.num_seqs, H = v.num_heads;
  if (c->attend_tiled) {
    const int64_t size = kv_size(c->type);
    auto bytes = [&](const KvPool& q) {
      return KvBytes{static_cast<uint32_t>(q.page * size), static_cast<uint32_t>(q.slot * size), static_cast<uint32_t>(q.head * size)};
    };
    p.kb = bytes(v.k);
    p.vb = bytes(v.v);
    p.same = p.kb.page == p.vb.page && p.kb.slot == p.vb.slot && p.kb.head == p.vb.head;
    WB_TRY(by_shape(v, c->type, [&](auto g, auto* kernel) {
      using G = decltype(g);
      p.cluster = c->attend_cluster;
      const int blocks = p.cluster > 0 ? v.num_seqs * v.num_kv * p.head_groups * p.cluster : c->attend_blocks;
      WB_TRY(launch_after(kernel, dim3(blocks), G::kThreads, G::kSmem, st, p, p.cluster));
      // a unit of one tile is never cut
      if ((p.cluster > 0 || v.max_slots <= G::kKeys) && !a.accumulate) return Status::Ok();
      auto finish = [&](auto wide, auto warps) {
        constexpr int kW = decltype(warps)::value, kSlots = kW == 4 ? 1024 : 2048;  // slots of a block of weights
        const int chunks = a.accumulate ? std::min((v.max_slots + kSlots - 1) / kSlots, 64) : 0;
        return launch_after(k_attend_finish<static_cast<int>(G::kBias), decltype(wide)::value, kW>, dim3(H + v.num_kv * chunks, B), 32 * kW, 0, st, p);
      };
      const bool many = c->attend_blocks / p.head_groups > kManyParts * static_cast<int64_t>(v.num_seqs) * v.num_kv;
      auto by_parts = [&](auto wide) { return many ? finish(wide, std::integral_constant<int, 16>{}) : finish(wide, std::integral_constant<int, 4>{}); };
      return v.head_dim > 128 ? by_parts(std::true_type{}) : by_parts(std::false_type{});
    }));
  } else {
    p.splits = simple_splits(v);
    WB_TRY(by_type(c->type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      k_attend_simple<T><<<dim3(p.splits, H, B), 32 * kSimpleWarps, 0, st>>>(p);
      return cuda_status(cudaGetLastError(), "kv attend launch");
    }));
    k_attend_join<<<dim3(H, B), 128, 0, st>>>(p);
    if (a.accumulate) {
      const unsigned blocks = (v.max_slots + 255) / 256;
      k_attend_weights<<<dim3(blocks < 64 ? blocks : 64, v.num_kv, B), 256, 0, st>>>(p);
    }
  }
  return cuda_status(cudaGetLastError(), "kv attend launch");
}

} // namespace wb
