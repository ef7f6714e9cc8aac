// gdense.cu -- matrix-vector products with 4-bit codes and group scales, and their quantiser (sm_100a).
#include "gdense.hpp"

#include "codec.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace wb {
namespace {

__device__ __forceinline__ float scale_value(uint16_t bits, int type) {
  return type == kScaleF16 ? __half2float(__ushort_as_half(bits)) : __bfloat162float(__ushort_as_bfloat16(bits));
}

// ---------------------------------------------------------------- layout
//
// The weights are cut into row groups of 16 outputs and chunks of 256 inputs; a record holds one
// row group's chunk: for each unit of 64 inputs 512 bytes of codes (lane l's 16 bytes are its A
// fragments of the unit's four m16n8k16 MMAs), then 16 scales and, for Uint4, 16 zero points
// per set of sg inputs ([8 rows][set][row, row + 8]), sg being the largest of 32, 64, 128, 256 that
// divides the group. Records of a row group follow one another, so a warp's piece of work is one
// contiguous copy. The inputs' order within a unit is the MMAs' own: input 32 (j / 2) + 8 t +
// 4 (j % 2) + 2 r + e is element e of register r of block j in lane t, so that 8 consecutive inputs
// of x are a lane's B fragments of two blocks, which span 32 inputs.
constexpr int kChunk = 256, kUnit = 64;

// BFloat16 scales of which some are 2^96 or more; their records keep sets of 32 inputs, so that this
// rare kind needs one width of set only.
constexpr int kScaleLarge = 4;

struct Layout {
  int row_groups, chunks, units;  // units of 64 inputs in all
  int sg, sets;                   // inputs of a scale set, sets of a record
  int tail;                       // bytes of a record's scales and zero points
  int64_t group_bytes;            // records of a row group
};

Layout layout_of(int rows, int cols, int group, int code, int scale_type) {
  Layout l;
  l.row_groups = (rows + 15) / 16;
  l.units = (cols + kUnit - 1) / kUnit;
  l.chunks = (cols + kChunk - 1) / kChunk;
  l.sg = scale_type == kScaleLarge ? 32 : group % 256 == 0 ? 256 : (group % 128 == 0 ? 128 : (group % 64 == 0 ? 64 : 32));
  l.sets = kChunk / l.sg;
  l.tail = l.sets * (code == kCodeUint4 ? 48 : 32);
  l.group_bytes = static_cast<int64_t>(l.units) * 512 + static_cast<int64_t>(l.chunks) * l.tail;
  return l;
}

struct BuildArgs {
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zeros;
  int rows, cols, group, groups, code;
  Layout l;
  uint8_t* out;
};

// One block per record.
__global__ void __launch_bounds__(128) k_group_build(const __grid_constant__ BuildArgs a) {
  const int chunk = blockIdx.x % a.l.chunks, rg = blockIdx.x / a.l.chunks;
  const int units = min(kChunk / kUnit, a.l.units - chunk * (kChunk / kUnit));
  uint8_t* rec = a.out + rg * a.l.group_bytes + static_cast<int64_t>(chunk) * (2048 + a.l.tail);
  const int64_t row_bytes = (a.cols + 1) / 2;
  for (int i = threadIdx.x; i < units * 128; i += blockDim.x) {  // 32-bit words of codes
    const int unit = i >> 7, lane = (i >> 2) & 31, j = i & 3, g = lane >> 2, t = lane & 3;
    uint32_t word = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // A register r: row g + 8 (r & 1), inputs + 2 (r >> 1)
      const int o = rg * 16 + g + 8 * (r & 1);
      const int k = chunk * kChunk + unit * kUnit + 32 * (j >> 1) + 8 * t + 4 * (j & 1) + 2 * (r >> 1);
      uint32_t two = 0;
      if (o < a.rows && k < a.cols) {
        two = a.codes[o * row_bytes + k / 2];
        if (k + 1 >= a.cols) two &= 15u;
        // Int4 is kept with its sign bit flipped: the code is the value plus 8
        if (a.code == kCodeInt4) two ^= k + 1 >= a.cols ? 0x08u : 0x88u;
      }
      if (a.code == kCodeFp4) word |= two << (8 * r);
      else word |= (two & 15u) << (4 * r) | (two >> 4) << (4 * r + 16);
    }
    *reinterpret_cast<uint32_t*>(rec + unit * 512 + lane * 16 + j * 4) = word;
  }
  uint16_t* sc = reinterpret_cast<uint16_t*>(rec + units * 512);
  uint8_t* zp = rec + units * 512 + a.l.sets * 32;
  for (int i = threadIdx.x; i < a.l.sets * 16; i += blockDim.x) {  // [g][set][2]: rows g, g + 8
    const int g = i / (2 * a.l.sets), set = (i >> 1) % a.l.sets, o = rg * 16 + g + 8 * (i & 1);
    const int k = chunk * kChunk + set * a.l.sg;
    const bool ok = o < a.rows && k < a.cols;
    const int64_t at = static_cast<int64_t>(o) * a.groups + k / a.group;
    sc[i] = ok ? a.scales[at] : 0;
    if (a.code == kCodeUint4) zp[i] = ok ? a.zeros[at] : 0;
  }
}

// *large = 1 if a finite BFloat16 scale is 2^96 or more.
__global__ void k_group_scales(const uint16_t* scales, int64_t n, int* large) {
  bool any = false;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int e = (scales[i] >> 7) & 255;
    any = any || (e >= 127 + 96 && e < 255);
  }
  if (__any_sync(0xffffffffu, any) && (threadIdx.x & 31) == 0) *large = 1;
}

// ---------------------------------------------------------------- matrix-vector product
//
// HBM bound: in * out / 2 bytes of codes and 2 (Uint4: 3) bytes per group of scales are read once,
// for 2 in out flops per token. A warp loads a record straight into registers, in fragment order,
// one record ahead of the one it multiplies on the register path of the tensor cores: codes become
// exact f16 A fragments, x is two f16 parts (22 bits) after scaling each token's chunk by a power
// of two, part p of token b in column 2 b + p, so that a thread's pair of accumulators is one
// token. Products are exact; a scale set's sum (fp32, at most 256 products) is multiplied by its
// scale and added to the row's fp32 sum. (Records copied to rings of shared memory by the bulk
// engine, 8 warps a block, were slower on layers below 100 MB: the ring leaves half the warps.)
// Measured at one token: FP4, 16384 -> 65536, groups of 32 (0.6 GB), 107 to 112 us by the GPU and its
// power cap, 5.4 to 5.7 TB/s (82 to 86 % of a copy); Int4, 4096 -> 4096, groups of 128 (8.7 MB), 5.2 us,
// of which 1.3 are the bytes and the rest launch, prologue, one pass of loads and the blocks' join (8.2
// at eight tokens: each block makes its own f16 parts of x); Int4, 16384 -> 65536, groups of 128: 102 to
// 109, 112 to 118 and 146 to 157 us at 1, 4 and 8 tokens (the second tile of tokens doubles the MMAs);
// Uint4, groups of 64, 114 to 120 us at one.
// tcgen05 needs N >= 8 and M = 128 rows of dequantised weights in shared or tensor memory; at 1..8
// tokens the conversion is the work, and the register path takes its result without a store.
//
// The records (row group by row group, chunk by chunk) are cut into equal runs. Layers that give
// every warp a row group or more make the runs the warps', which then never wait for one another;
// smaller ones make them the blocks', whose warps take every 16th record and leave their sums in
// shared memory, where those of up to eight row groups are added and finished together. Row groups
// that a run's ends cut are joined through global memory by the last run to come, in run order;
// small layers avoid that with runs of whole row groups. The first weight loads start before the
// previous kernel's end is waited for.
constexpr int kMaxTokens = 8;
constexpr int kGWarps = 16;
constexpr int kGThreads = 32 * kGWarps;
constexpr int kXBytes = 140 * 1024;  // shared memory for x
constexpr int kHold = 8;             // row groups whose sums wait in shared memory for one barrier

struct GArgs {
  const uint8_t* w;
  Layout l;
  const double* bias;
  int rows, cols, act, bias_len;
  const float* x;
  int64_t x_ld;
  float* pre;
  float* post;
  int n;             // tokens, 1..8
  int slabs;         // parts of the inputs whose x fits shared memory, each with its own blocks
  int slab_chunks;   // chunks of a slab (the last one may have fewer)
  int slab_blocks;   // blocks of a slab
  int solo;          // runs are the warps', not the blocks'
  int aligned;       // (blocks') runs are whole row groups
  float* part;       // [runs][2][16][8]
  int* tickets;      // [slabs][row groups], zero between calls
  float* slab_sum;   // [slabs][n][rows], with more than one slab
};

__device__ __forceinline__ void g_write(const GArgs& a, int o, int b, float y) {
  double v = static_cast<double>(y);
  if (o < a.bias_len) v += a.bias[o];
  const int64_t at = static_cast<int64_t>(b) * a.rows + o;
  if (a.pre) a.pre[at] = static_cast<float>(v);
  a.post[at] = static_cast<float>(activate(a.act, v));
}

__device__ __forceinline__ void g_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void g_mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// A fragment of one block: E2M1 bytes through the converter; integer codes n as the f16 1024 + n
// (or 1024 + 16 n, where the nibble stands four bits higher), minus 1024 + zero (or times 1/16,
// minus 64 + zero), both exact. That f16 numbers of exponent 10 hold an integer in their last bits, so
// that an OR converts it, is the published way (Kim, Henry, Fahim, Hassan Awadalla, "Who Says Elephants
// Can't Run", 2022); the constants follow from the format.
template <int kCode>
__device__ __forceinline__ void g_decode(uint32_t w, __half2 z0, __half2 z1, uint32_t (&a)[4]) {
  if constexpr (kCode == kCodeFp4) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(w));
  } else {
    const uint32_t v = w >> 8;
    // (x & mask) | 0x6400: one three-input operation
    auto code = [](uint32_t x, uint32_t mask) {
      uint32_t y;
      asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(mask), "r"(0x64006400u));
      return *reinterpret_cast<__half2*>(&y);
    };
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const __half2 r0 = __hsub2(code(w, 0x000f000fu), z0);
    const __half2 r1 = __hfma2(code(w, 0x00f000f0u), sixteenth, z1);
    const __half2 r2 = __hsub2(code(v, 0x000f000fu), z0);
    const __half2 r3 = __hfma2(code(v, 0x00f000f0u), sixteenth, z1);
    a[0] = *reinterpret_cast<const uint32_t*>(&r0);
    a[1] = *reinterpret_cast<const uint32_t*>(&r1);
    a[2] = *reinterpret_cast<const uint32_t*>(&r2);
    a[3] = *reinterpret_cast<const uint32_t*>(&r3);
  }
}

__device__ __forceinline__ uint4 ld_weights(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// A lane's share of a record: its codes of the four units, and the scales and zero points of rows g
// and g + 8 for each set of kSub inputs.
template <int kCode, int kSub>
struct GRecord {
  static constexpr int kSets = kChunk / kSub;
  uint4 codes[4];
  uint32_t scales[kSets];
  uint32_t zeros[kCode == kCodeUint4 ? (kSets + 1) / 2 : 1];  // two sets a word
};

// The words of kN sets that lie together.
template <int kN>
__device__ __forceinline__ void ld_words(const uint8_t* p, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < kN; i += 4) {
    if constexpr (kN >= 4) asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "l"(p + 4 * i));
    else if constexpr (kN == 2) asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    else asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  }
}

// kNT n8 tiles of tokens (1: up to 4 tokens, 2: up to 8). kSub: inputs of a scale set (32, 64, 128
// or 256). kScale: the scales' kind (kScaleF16, kScaleBF16 or kScaleLarge).
template <int kCode, int kNT, int kSub, int kScale>
__global__ void __launch_bounds__(kGThreads, 1) k_group_gemv(const __grid_constant__ GArgs a) {
  using Record = GRecord<kCode, kSub>;
  extern __shared__ __align__(128) uint8_t sx[];  // x parts: [2 n columns][slab inputs] f16
  __shared__ __align__(16) uint8_t s_zero[kChunk * 2];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  const int slab = blockIdx.x / a.slab_blocks, rank = blockIdx.x - slab * a.slab_blocks;
  const int c_first = slab * a.slab_chunks, chunks = min(a.slab_chunks, a.l.chunks - c_first);
  const int pitch = a.slab_chunks * (kChunk * 2) + 64;  // bytes of a column; two columns fill the banks
  float* const sxs = reinterpret_cast<float*>(sx + 2 * a.n * pitch);  // [token][chunk] 2^-e
  constexpr int kOuts = 16 * 4 * kNT;  // sums of a row group: [row][token]
  float* const s_red = sxs + (a.n * a.slab_chunks + 3) / 4 * 4;  // [kHold][warp][kOuts], not with runs of the warps

  asm volatile("griddepcontrol.launch_dependents;");
  // this block's or this warp's run of records, and the warp's share of it: every step-th from first_rec
  const int total = a.l.row_groups * chunks;
  const int runs = a.solo ? a.slab_blocks * kGWarps : a.slab_blocks, run = a.solo ? rank * kGWarps + w : rank;
  auto run_start = [&](int i) {
    return a.aligned ? static_cast<int>(static_cast<int64_t>(i) * a.l.row_groups / runs) * chunks
                     : static_cast<int>(static_cast<int64_t>(i) * total / runs);
  };
  const int r0 = run_start(run), r1 = run_start(run + 1);
  const int step = a.solo ? 1 : kGWarps;
  const int first_rec = a.solo ? r0 : r0 + w;

  // loads, one record ahead
  const int rec_bytes = 2048 + a.l.tail, last_units = a.l.units - (a.l.chunks - 1) * (kChunk / kUnit);
  const int to_last = last_units < kChunk / kUnit ? a.l.chunks - 1 - c_first : -1;  // the chunk that is short
  int rg = first_rec / chunks, ch = first_rec - rg * chunks;
  const uint8_t* src = a.w + rg * a.l.group_bytes + static_cast<int64_t>(c_first + ch) * rec_bytes + lane * 16;
  const int step_bytes = step * rec_bytes, to_scales = g * (4 * Record::kSets) - lane * 16, to_zeros = 32 * Record::kSets + g * (2 * Record::kSets) - lane * 16;
  int loaded = first_rec;
  auto load = [&](Record& r) {
    if (loaded >= r1) return;
    const uint8_t* tl = src + 2048;
    if (ch != to_last) {
#pragma unroll
      for (int u = 0; u < kChunk / kUnit; ++u) r.codes[u] = ld_weights(src + u * 512);
    } else {  // codes of absent units are zero; their x is zero too
#pragma unroll
      for (int u = 0; u < kChunk / kUnit; ++u) r.codes[u] = u < last_units ? ld_weights(src + u * 512) : make_uint4(0, 0, 0, 0);
      tl = src + last_units * 512;
    }
    ld_words<Record::kSets>(tl + to_scales, r.scales);
    if constexpr (kCode == kCodeUint4) {
      if constexpr (Record::kSets == 1) r.zeros[0] = *reinterpret_cast<const uint16_t*>(tl + to_zeros);
      else ld_words<Record::kSets / 2>(tl + to_zeros, r.zeros);
    }
    loaded += step;
    ch += step;
    src += step_bytes;
    if (ch >= chunks) {
      do {
        ch -= chunks;
        ++rg;
      } while (ch >= chunks);
      src = a.w + rg * a.l.group_bytes + static_cast<int64_t>(c_first + ch) * rec_bytes + lane * 16;
    }
  };
  Record rec_a, rec_b;  // in turn the one at work and the one ahead
  load(rec_a);
  if (tid < kChunk / 8) *reinterpret_cast<uint4*>(s_zero + 16 * tid) = make_uint4(0, 0, 0, 0);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  // x: a warp takes a token's chunk at a time, eight inputs a lane
  const bool vec = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (a.x_ld & 3) == 0;
  const bool vec2 = (reinterpret_cast<uintptr_t>(a.x) & 7) == 0 && (a.x_ld & 1) == 0;
  constexpr int kFly = 4;  // chunks whose loads are in flight together (8: more code to fetch cold, 8 tokens 8.2 -> 8.5 us)
  const int b_step = kGWarps / chunks, c_step = kGWarps - b_step * chunks;
  auto advance = [&](int& b, int& c) {
    b += b_step;
    c += c_step;
    if (c >= chunks) {
      c -= chunks;
      ++b;
    }
  };
  for (int b0 = w / chunks, c0 = w - b0 * chunks; b0 < a.n;) {
    float v[kFly][8];
    int b = b0, c = c0;
#pragma unroll
    for (int y = 0; y < kFly; ++y) {
      const int k0 = (c_first + c) * kChunk + 8 * lane;
      const float* xs = a.x + b * a.x_ld + k0;
      const bool on = b < a.n;
      if (vec && on && k0 + 8 <= a.cols) {
        *reinterpret_cast<float4*>(v[y]) = ld_dep4(xs);
        *reinterpret_cast<float4*>(v[y] + 4) = ld_dep4(xs + 4);
      } else if (vec2 && on && k0 + 8 <= a.cols) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(v[y][e]), "=f"(v[y][e + 1]) : "l"(xs + e));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[y][e] = on && k0 + e < a.cols ? ld_dep(xs + e) : 0.0f;
      }
      advance(b, c);
    }
#pragma unroll
    for (int y = 0; y < kFly; ++y) {
      if (b0 >= a.n) break;
      // the chunk's largest finite |x| goes to [2^14, 2^15)
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[y][e]) & 0x7fffffffu);
      top = __reduce_max_sync(0xffffffffu, top);
      const bool finite = top < 0x7f800000u;
      if (!finite) {
        top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, isfinite(v[y][e]) ? __float_as_uint(v[y][e]) & 0x7fffffffu : 0u);
        top = __reduce_max_sync(0xffffffffu, top);
      }
      const int ex = min(126, 141 - static_cast<int>(top >> 23));
      const float f = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);  // 2^ex
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = v[y][2 * e] * f, q = v[y][2 * e + 1] * f;
        const __half2 h = __floats2half2_rn(p, q);
        const float2 r = __half22float2(h);
        float dp = p - r.x, dq = q - r.y;
        if (!finite) {  // infinities and NaN stay in the first part
          dp = isfinite(p) ? dp : 0.0f;
          dq = isfinite(q) ? dq : 0.0f;
        }
        const __half2 l = __floats2half2_rn(dp, dq);
        hi[e] = *reinterpret_cast<const uint32_t*>(&h);
        lo[e] = *reinterpret_cast<const uint32_t*>(&l);
      }
      uint8_t* dst = sx + 2 * b0 * pitch + (c0 * kChunk + 8 * lane) * 2;
      *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(dst + pitch) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      if (lane == 0) sxs[b0 * a.slab_chunks + c0] = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
      advance(b0, c0);
    }
  }
  __syncthreads();

  // columns without a token read zeros
  const uint8_t* xcol[kNT];
  int xstep[kNT];
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
    const bool on = 8 * nt + g < 2 * a.n;
    xcol[nt] = on ? sx + (8 * nt + g) * pitch + 16 * t : s_zero + 16 * t;
    xstep[nt] = on ? kChunk * 2 : 0;
  }
  float acc[kNT][4];
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;

  auto write = [&](int rs, int r, int b, float v) {
    const int o = rs * 16 + r;
    if (o >= a.rows) return;
    if (a.slabs == 1) g_write(a, o, b, v);
    else a.slab_sum[(static_cast<int64_t>(slab) * a.n + b) * a.rows + o] = v;
  };
  // The runs that cut a row group leave their sums; the last one to come adds them in run order. A
  // run has two slots: the second for a row group that begins in it, the first for one that goes on.
  constexpr int kSlot = 16 * kMaxTokens;
  auto run_of = [&](int rec) { return static_cast<int>((static_cast<int64_t>(rec + 1) * runs - 1) / total); };
  auto slot_of = [&](int begin) { return a.part + (2 * (static_cast<int64_t>(slab) * runs + run) + (begin >= r0 ? 1 : 0)) * kSlot; };
  auto ticket_of = [&](int rs) { return a.tickets + static_cast<int64_t>(slab) * a.l.row_groups + rs; };
  auto joined = [&](int begin, int i) {
    const int run0 = run_of(begin), run1 = run_of(begin + chunks - 1);
    const float* cut = a.part + 2 * (static_cast<int64_t>(slab) * runs + run0) * kSlot + i;
    float v = __ldcg(cut + kSlot);
    for (int x = 1; x <= run1 - run0; ++x) v += __ldcg(cut + 2ll * x * kSlot);
    return v;
  };
  int held = 0;          // row groups in s_red
  int next = first_rec;  // the warp's next record
  bool turn = false;
  int rs = r0 / chunks;
  for (int seg = r0; seg < r1; ++rs) {  // row groups of the run
    const int set_begin = rs * chunks, set_end = set_begin + chunks, end = min(set_end, r1);
    const bool whole = seg == set_begin && end == set_end;
    auto record = [&](const Record& r, Record& ahead) {
      const int c = next - set_begin;
      load(ahead);
      const uint8_t* xp[kNT];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) xp[nt] = xcol[nt] + c * xstep[nt];
      float sum[kNT][4];  // the record's, in units of the thread's token's xs
      float part[kNT][4];
      // The power of two that x was multiplied by is undone after the scales, which carry no sum (below
      // 2^31) past the largest float while they are below 2^96. With larger ones (kScaleLarge) as much
      // of a small x's power as keeps sums below 1 is undone before them, or a result that is finite
      // would pass through an infinity. (Done for all BFloat16 scales, 8 tokens take a tenth longer.)
      constexpr float kLeast = 0x1p-32f;
      auto undo = [&](int nt) { return 4 * nt + t < a.n ? sxs[(4 * nt + t) * a.slab_chunks + c] : 0.0f; };
      float xa[kNT];
      if constexpr (kScale == kScaleLarge) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) xa[nt] = fminf(fmaxf(undo(nt), kLeast), 1.0f);
      }
#pragma unroll
      for (int u = 0; u < kChunk / kUnit; ++u) {
        uint4 xb[kNT][2];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const uint4* xs = reinterpret_cast<const uint4*>(xp[nt] + u * (kUnit * 2));
          xb[nt][0] = xs[0];
          xb[nt][1] = xs[4];
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // halves of the unit
          constexpr int kS = kSub;
          const int k = u * kUnit + 32 * hf, set = k / kS;  // constants once unrolled
          const bool begins = k % kS == 0, ends = (k + 32) % kS == 0;
          __half2 z0 = __float2half2_rn(1032.0f), z1 = __float2half2_rn(-72.0f);
          if constexpr (kCode == kCodeUint4) {
            const uint32_t z = r.zeros[set >> 1] >> (16 * (set & 1));
            z0 = __half2half2(__ushort_as_half(static_cast<unsigned short>(0x6400u | (z & 0xffu))));
            z1 = __hneg2(__half2half2(__ushort2half_rn(static_cast<unsigned short>(64u + ((z >> 8) & 0xffu)))));
          }
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const int j = 2 * hf + jj;
            const uint32_t word = j == 0 ? r.codes[u].x : (j == 1 ? r.codes[u].y : (j == 2 ? r.codes[u].z : r.codes[u].w));
            uint32_t fr[4];
            g_decode<kCode>(word, z0, z1, fr);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              const uint4 x = xb[nt][hf];
              const uint32_t b0 = jj ? x.z : x.x, b1 = jj ? x.w : x.y;
              if (jj == 0 && begins) g_mma0(part[nt], fr, b0, b1);
              else g_mma(part[nt], fr, b0, b1);
            }
          }
          if (ends) {
            const uint32_t s2 = r.scales[set];
            const float s0 = scale_value(static_cast<uint16_t>(s2), kScale), s1 = scale_value(static_cast<uint16_t>(s2 >> 16), kScale);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if constexpr (kScale == kScaleLarge) part[nt][e] *= xa[nt];
                sum[nt][e] = (set == 0 ? 0.0f : sum[nt][e]) + part[nt][e] * (e < 2 ? s0 : s1);
              }
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float xs = undo(nt);
        if constexpr (kScale == kScaleLarge) xs = xs > 1.0f ? xs : (xs < kLeast ? xs * (1.0f / kLeast) : 1.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] += sum[nt][e] * xs;
      }
    };
    for (; next < end; next += step) {
      if (turn) record(rec_b, rec_a);
      else record(rec_a, rec_b);
      turn = !turn;
    }
    if (a.solo) {
      bool last = true;
      if (!whole) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) slot_of(set_begin)[(g + 8 * e) * kMaxTokens + 4 * nt + t] = acc[nt][2 * e] + acc[nt][2 * e + 1];
        __syncwarp();
        int before = 0;
        if (lane == 0) {
          __threadfence();
          before = atomicAdd(ticket_of(rs), 1);
        }
        last = __shfl_sync(0xffffffffu, before, 0) == run_of(set_end - 1) - run_of(set_begin);
        if (last) {
          __threadfence();
          if (lane == 0) *ticket_of(rs) = 0;
        }
      }
      if (last) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = g + 8 * e, b = 4 * nt + t;
            if (b < a.n) write(rs, r, b, whole ? acc[nt][2 * e] + acc[nt][2 * e + 1] : joined(set_begin, r * kMaxTokens + b));
          }
      }
    } else {
      float* const to = s_red + (held * kGWarps + w) * kOuts;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) to[(g + 8 * e) * (4 * kNT) + 4 * nt + t] = acc[nt][2 * e] + acc[nt][2 * e + 1];
      if (++held == kHold || end == r1) {
        // add the warps' sums of the row groups held, finish those that are whole
        __syncthreads();
        const int first_rs = rs + 1 - held;
        for (int i = tid; i < held * kOuts; i += kGThreads) {
          const int x = i / kOuts, at = i - x * kOuts, r = at / (4 * kNT), b = at - r * (4 * kNT);
          if (b >= a.n) continue;
          float v = 0.0f;
#pragma unroll
          for (int y = 0; y < kGWarps; ++y) v += s_red[(x * kGWarps + y) * kOuts + at];
          const int begin = (first_rs + x) * chunks;
          if (begin >= r0 && begin + chunks <= r1) write(first_rs + x, r, b, v);
          else slot_of(begin)[r * kMaxTokens + b] = v;
        }
        // at most the first and the last row group of the run are cut
        for (int x = 0; x < held; ++x) {
          const int cut_rs = first_rs + x, begin = cut_rs * chunks;
          if (begin >= r0 && begin + chunks <= r1) continue;
          __syncthreads();
          if (tid == 0) {
            __threadfence();
            s_last = atomicAdd(ticket_of(cut_rs), 1) == run_of(begin + chunks - 1) - run_of(begin);
          }
          __syncthreads();
          if (s_last) {
            __threadfence();
            if (tid == 0) *ticket_of(cut_rs) = 0;
            const int r = tid & 15, b = tid >> 4;
            if (b < a.n) write(cut_rs, r, b, joined(begin, r * kMaxTokens + b));
          }
        }
        held = 0;
        if (end < r1) __syncthreads();  // before the next sums are left there
      }
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
    seg = end;
  }
}

// y from the slabs' sums, in slab order: 4 bytes a slab and output, from L2.
__global__ void __launch_bounds__(256) k_group_slabs(const __grid_constant__ GArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int o = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (o >= a.rows) return;
  float v = 0.0f;
  for (int s = 0; s < a.slabs; ++s) v += __ldcg(a.slab_sum + (static_cast<int64_t>(s) * a.n + b) * a.rows + o);
  g_write(a, o, b, v);
}

// The quantiser, run once per matrix: 16384 x 16384 in groups of 64 (1.07 GB read) take 1.03 ms (Int4),
// 1.14 (Uint4) and 1.59 (FP4), a sixth of a copy's rate, bound by a division per weight and the few
// loads that a warp has in flight. One warp per (row, group): the group's range gives its scale, rounded
// to the scale's type before the codes are chosen, so that decoding multiplies by what the codes were
// divided by. A group that holds an infinity or NaN gets a NaN scale: its row says so, where codes would
// hide it.
template <int kCode>
__global__ void __launch_bounds__(256)
    k_group_quantize(const float* __restrict__ W, int rows, int cols, int group, int groups, int scale_type, uint8_t* codes,
                     uint16_t* scales, uint8_t* zeros) {
  const int64_t unit = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (unit >= static_cast<int64_t>(rows) * groups) return;
  const int o = static_cast<int>(unit / groups), g = static_cast<int>(unit - static_cast<int64_t>(o) * groups);
  const float* w = W + static_cast<int64_t>(o) * cols;
  const int k0 = g * group, k1 = k0 + group < cols ? k0 + group : cols;
  float lo = 0.0f, hi = 0.0f;  // zero stays representable
  bool finite = true;
  for (int k = k0 + lane; k < k1; k += 32) {
    lo = fminf(lo, w[k]);
    hi = fmaxf(hi, w[k]);
    finite = finite && isfinite(w[k]);
  }
  finite = __all_sync(0xffffffffu, finite);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  const float amax = fmaxf(-lo, hi);
  float s = kCode == kCodeFp4 ? amax / 6.0f : (kCode == kCodeInt4 ? amax / 7.0f : (hi - lo) / 15.0f);
  uint16_t bits;
  if (scale_type == kScaleF16) bits = __half_as_ushort(__float2half_rn(fminf(s, 65504.0f)));
  else bits = __bfloat16_as_ushort(__float2bfloat16_rn(fminf(s, 3.3895314e38f)));
  if (!finite) bits = scale_type == kScaleF16 ? 0x7e00u : 0x7fc0u;
  s = scale_value(bits, scale_type);
  const float zero = kCode == kCodeUint4 && s > 0.0f ? fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f) : 0.0f;
  if (lane == 0) {
    scales[unit] = bits;
    if (kCode == kCodeUint4) zeros[unit] = static_cast<uint8_t>(zero);
  }
  const int bytes = (cols + 1) / 2;
  for (int i = k0 / 2 + lane; i < (k1 + 1) / 2; i += 32) {
    uint32_t two = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = 2 * i + e;
      const float v = k < k1 && s > 0.0f ? w[k] / s : 0.0f;
      uint32_t c;
      if (kCode == kCodeFp4) c = enc_fp4(fminf(fmaxf(v, -6.0f), 6.0f));
      else if (kCode == kCodeInt4) c = static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(v), -8.0f), 7.0f))) & 15u;
      else c = static_cast<uint32_t>(fminf(fmaxf(rintf(v) + zero, 0.0f), 15.0f));
      if (k >= k1) c = 0;
      two |= c << (4 * e);
    }
    codes[static_cast<int64_t>(o) * bytes + i] = static_cast<uint8_t>(two);
  }
}

} // namespace

GroupDense::~GroupDense() {
  cudaSetDevice(device);
  for (void* p : {static_cast<void*>(w), static_cast<void*>(bias), static_cast<void*>(work)})
    if (p) cudaFree(p);
}

namespace {

struct GPlan {
  int slabs, slab_chunks, slab_blocks, solo, aligned, smem;
};

GPlan plan_of(int sms, const Layout& l, int n) {
  GPlan p;
  const int fit = (kXBytes - 2 * n * 64) / (n * (2 * kChunk * 2 + 4));  // chunks of x in shared memory
  p.slabs = (l.chunks + fit - 1) / fit;
  p.slab_chunks = (l.chunks + p.slabs - 1) / p.slabs;
  p.slabs = (l.chunks + p.slab_chunks - 1) / p.slab_chunks;
  // every warp of a block has a record or more
  const int64_t last = l.chunks - (p.slabs - 1) * p.slab_chunks;
  const int64_t most = std::max<int64_t>(1, l.row_groups * last / kGWarps);
  p.slab_blocks = static_cast<int>(std::min<int64_t>(std::max(1, sms / p.slabs), most));
  p.solo = l.row_groups >= p.slab_blocks * kGWarps;
  p.aligned = 0;
  p.smem = 2 * n * (p.slab_chunks * kChunk * 2 + 64) + (n * p.slab_chunks + 3) / 4 * 16;
  if (!p.solo) {
    p.smem += kHold * kGWarps * 16 * (n > 4 ? 8 : 4) * 4;
    // Whole row groups leave blocks idle for part of the last round, runs that cut them pay a join at
    // their end. Measured at one token, whole and cut: 19 MB of records missed by idle blocks (4800 x
    // 16384) 13.6 and 14.7 us, 20 MB (9504 x 16384) 20.0 and 20.9, 25 MB (2400 x 20480) 12.9 and 12.4,
    // 39 MB (2400 x 32768) 17.8 and 15.9.
    const int per = (l.row_groups + p.slab_blocks - 1) / p.slab_blocks;
    const double idle = static_cast<double>(per) * p.slab_blocks / l.row_groups - 1.0;
    p.aligned = l.row_groups >= p.slab_blocks && idle * l.group_bytes * l.row_groups < 22e6;
    // Fewer row groups than blocks: one a block, unless it is long. One a block and cut: 135 KB (1024 x
    // 16384) 6.8 and 10.0 us, 270 KB (1024 x 32768) 11.5 and 12.9, with half the row groups (512 x 32768)
    // 11.4 and 11.4.
    if (l.row_groups < p.slab_blocks && l.group_bytes < 300e3) {
      p.slab_blocks = l.row_groups;
      p.aligned = 1;
    }
  }
  return p;
}

using GKernel = void (*)(GArgs);

template <int kSub, int kScale>
GKernel kernel_of(int code, int n) {
  if (code == kCodeFp4) return n > 4 ? k_group_gemv<kCodeFp4, 2, kSub, kScale> : k_group_gemv<kCodeFp4, 1, kSub, kScale>;
  if (code == kCodeInt4) return n > 4 ? k_group_gemv<kCodeInt4, 2, kSub, kScale> : k_group_gemv<kCodeInt4, 1, kSub, kScale>;
  return n > 4 ? k_group_gemv<kCodeUint4, 2, kSub, kScale> : k_group_gemv<kCodeUint4, 1, kSub, kScale>;
}

template <int kScale>
GKernel kernel_of(int sg, int code, int n) {
  return sg == 32 ? kernel_of<32, kScale>(code, n) : (sg == 64 ? kernel_of<64, kScale>(code, n) : (sg == 128 ? kernel_of<128, kScale>(code, n) : kernel_of<256, kScale>(code, n)));
}

GKernel kernel_of(const GroupDense& g, const Layout& l, int n) {
  if (g.scale_type == kScaleLarge) return kernel_of<32, kScaleLarge>(g.code, n);
  return g.scale_type == kScaleF16 ? kernel_of<kScaleF16>(l.sg, g.code, n) : kernel_of<kScaleBF16>(l.sg, g.code, n);
}

template <typename K>
Status g_launch(K* kernel, dim3 grid, int threads, int smem, cudaStream_t st, const GArgs& a) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a), "group gemv launch");
}

// Device copies of a mount's host arrays, freed when the mount is done.
struct Staged {
  void* p = nullptr;
  ~Staged() { if (p) cudaFree(p); }
  Status put(const void* src, size_t n) {
    WB_CUDA(cudaMalloc(&p, n));
    return cuda_status(cudaMemcpy(p, src, n, cudaMemcpyHostToDevice), "group dense h2d");
  }
};

Status gdense_fill(GroupDense* g, const GroupDenseSrc& src) {
  WB_CUDA(cudaSetDevice(g->device));
  WB_CUDA(cudaDeviceGetAttribute(&g->sms, cudaDevAttrMultiProcessorCount, g->device));
  const size_t n_codes = static_cast<size_t>(g->rows) * ((g->cols + 1) / 2), n_groups = static_cast<size_t>(g->rows) * g->groups;
  BuildArgs b;
  b.codes = src.codes;
  b.scales = static_cast<const uint16_t*>(src.scales);
  b.zeros = src.zeros;
  Staged codes, scales, zeros;
  if (!src.on_device) {
    WB_TRY(codes.put(src.codes, n_codes));
    WB_TRY(scales.put(src.scales, n_groups * 2));
    b.codes = static_cast<const uint8_t*>(codes.p);
    b.scales = static_cast<const uint16_t*>(scales.p);
    if (src.zeros) {
      WB_TRY(zeros.put(src.zeros, n_groups));
      b.zeros = static_cast<const uint8_t*>(zeros.p);
    }
  }
  b.rows = g->rows;
  b.cols = g->cols;
  b.group = g->group;
  b.groups = g->groups;
  b.code = g->code;
  if (g->scale_type == kScaleBF16) {
    Staged large;
    int any = 0;
    WB_TRY(large.put(&any, sizeof any));
    k_group_scales<<<static_cast<unsigned>(std::min<size_t>((n_groups + 255) / 256, 4 * g->sms)), 256>>>(b.scales, n_groups, static_cast<int*>(large.p));
    WB_CUDA(cudaGetLastError());
    WB_CUDA(cudaMemcpy(&any, large.p, sizeof any, cudaMemcpyDeviceToHost));
    if (any) g->scale_type = kScaleLarge;
  }
  b.l = layout_of(g->rows, g->cols, g->group, g->code, g->scale_type);
  WB_CUDA(cudaMalloc(&g->w, b.l.group_bytes * b.l.row_groups));
  b.out = g->w;
  k_group_build<<<static_cast<unsigned>(static_cast<int64_t>(b.l.row_groups) * b.l.chunks), 128>>>(b);
  WB_CUDA(cudaGetLastError());
  g->bias_len = static_cast<int>(std::min<size_t>(src.bias_len, g->rows));
  if (g->bias_len > 0) {
    WB_CUDA(cudaMalloc(&g->bias, static_cast<size_t>(g->bias_len) * 8));
    WB_CUDA(cudaMemcpy(g->bias, src.bias, static_cast<size_t>(g->bias_len) * 8, cudaMemcpyHostToDevice));
  }
  // workspaces for every number of tokens
  size_t part = 0, tickets = 0, slabs = 0;
  for (int n = 1; n <= kMaxTokens; ++n) {
    const GPlan p = plan_of(g->sms, b.l, n);
    part = std::max<size_t>(part, static_cast<size_t>(p.slabs) * p.slab_blocks * (p.solo ? kGWarps : 1) * 2 * 16 * kMaxTokens * 4);
    tickets = std::max<size_t>(tickets, static_cast<size_t>(p.slabs) * b.l.row_groups * 4);
    if (p.slabs > 1) slabs = std::max<size_t>(slabs, static_cast<size_t>(p.slabs) * n * g->rows * 4);
    WB_CUDA(cudaFuncSetAttribute(kernel_of(*g, b.l, n), cudaFuncAttributeMaxDynamicSharedMemorySize, kXBytes + kHold * kGWarps * 16 * 8 * 4 + 64));
  }
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  WB_CUDA(cudaMalloc(&g->work, up(tickets) + up(part) + up(slabs)));
  g->tickets = reinterpret_cast<int*>(g->work);
  g->part = reinterpret_cast<float*>(g->work + up(tickets));
  g->slab_sum = reinterpret_cast<float*>(g->work + up(tickets) + up(part));
  WB_CUDA(cudaMemset(g->work, 0, up(tickets)));
  return cuda_status(cudaDeviceSynchronize(), "group dense mount");
}

} // namespace

Status gdense_mount(int device, int rows, int cols, int group, int code, int scale_type, int act, const GroupDenseSrc& src,
                    GroupDense** out) {
  auto* g = new GroupDense();
  g->device = device;
  g->rows = rows;
  g->cols = cols;
  g->group = group;
  g->groups = (cols + group - 1) / group;
  g->code = code;
  g->scale_type = scale_type;
  g->act = act;
  const Status st = gdense_fill(g, src);
  if (!st.ok()) {
    cudaGetLastError();  // a failed allocation must not be taken for a later launch's error
    delete g;
    return st;
  }
  *out = g;
  return Status::Ok();
}

Status gdense_forward(GroupDense* g, int n, const float* x, int64_t x_ld, float* pre, float* post, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(g->device));
  GArgs a;
  a.w = g->w;
  a.l = layout_of(g->rows, g->cols, g->group, g->code, g->scale_type);
  a.bias = g->bias;
  a.rows = g->rows;
  a.cols = g->cols;
  a.act = g->act;
  a.bias_len = g->bias_len;
  a.x_ld = x_ld;
  a.part = g->part;
  a.tickets = g->tickets;
  a.slab_sum = g->slab_sum;
  for (int b = 0; b < n; b += kMaxTokens) {
    a.n = std::min(n - b, kMaxTokens);
    a.x = x + b * x_ld;
    a.pre = pre ? pre + static_cast<int64_t>(b) * g->rows : nullptr;
    a.post = post + static_cast<int64_t>(b) * g->rows;
    const GPlan p = plan_of(g->sms, a.l, a.n);
    a.slabs = p.slabs;
    a.slab_chunks = p.slab_chunks;
    a.slab_blocks = p.slab_blocks;
    a.solo = p.solo;
    a.aligned = p.aligned;
    WB_TRY(g_launch(kernel_of(*g, a.l, a.n), dim3(p.slabs * p.slab_blocks), kGThreads, p.smem, st, a));
    if (p.slabs > 1) WB_TRY(g_launch(k_group_slabs, dim3((g->rows + 255) / 256, a.n), 256, 0, st, a));
  }
  return Status::Ok();
}

int gdense_plan_values(int rows, int cols, int group, int code, int sms, int n, int64_t* out, int count) {
  const Layout l = layout_of(rows, cols, group, code, kScaleF16);
  const GPlan p = plan_of(sms, l, n);
  const int64_t runs = static_cast<int64_t>(p.slab_blocks) * (p.solo ? kGWarps : 1);
  // row groups that a run's end cuts, over all slabs
  int64_t cut = 0;
  for (int s = 0; s < p.slabs && !p.aligned; ++s) {
    const int64_t chunks = std::min(p.slab_chunks, l.chunks - s * p.slab_chunks), total = l.row_groups * chunks;
    int64_t last = -1;
    for (int64_t i = 1; i < runs; ++i) {
      const int64_t at = i * total / runs;
      if (at % chunks != 0 && at / chunks != last) {
        last = at / chunks;
        ++cut;
      }
    }
  }
  const int64_t values[] = {p.slabs, p.slab_chunks, p.slab_blocks, p.solo, p.aligned, p.smem, l.row_groups, l.chunks, runs, cut};
  constexpr int kValues = sizeof(values) / sizeof(values[0]);
  for (int i = 0; i < std::min(count, kValues); ++i) out[i] = values[i];
  return kValues;
}

Status group_quantize(int rows, int cols, int group, int code, int scale_type, const float* W, uint8_t* codes, void* scales,
                      uint8_t* zeros, cudaStream_t st) {
  const int groups = (cols + group - 1) / group;
  const int64_t units = static_cast<int64_t>(rows) * groups;
  const unsigned blocks = static_cast<unsigned>((units + 7) / 8);
  auto* s = static_cast<uint16_t*>(scales);
  if (code == kCodeFp4) k_group_quantize<kCodeFp4><<<blocks, 256, 0, st>>>(W, rows, cols, group, groups, scale_type, codes, s, zeros);
  else if (code == kCodeInt4) k_group_quantize<kCodeInt4><<<blocks, 256, 0, st>>>(W, rows, cols, group, groups, scale_type, codes, s, zeros);
  else k_group_quantize<kCodeUint4><<<blocks, 256, 0, st>>>(W, rows, cols, group, groups, scale_type, codes, s, zeros);
  return cuda_status(cudaGetLastError(), "group quantize launch");
}

} // namespace wb
