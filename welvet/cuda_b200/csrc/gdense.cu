// gdense.cu -- matrix-vector products with 4-bit codes and group scales, and their quantiser (sm_100a).
#include "gdense.hpp"

#include "codec.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace wb {
namespace {

__device__ __forceinline__ float scale_value(uint16_t bits, int type) {
  return type == kScaleF16 ? __half2float(__ushort_as_half(bits)) : __bfloat162float(__ushort_as_bfloat16(bits));
}

struct GArgs {
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zeros;
  const double* bias;
  int rows, cols, group, groups, scale_type, act, bias_len;
  const float* x;
  int64_t x_ld;
  float* pre;
  float* post;
  int n;
};

__device__ __forceinline__ void g_write(const GArgs& a, int o, int b, float y) {
  double v = static_cast<double>(y);
  if (o < a.bias_len) v += a.bias[o];
  const int64_t at = static_cast<int64_t>(b) * a.rows + o;
  if (a.pre) a.pre[at] = static_cast<float>(v);
  a.post[at] = static_cast<float>(activate(a.act, v));
}

constexpr int kMaxTokens = 8;

// A warp per output row: lanes over bytes of the row, the group's scale on every product, fp32 sums.
template <int kCode>
__global__ void __launch_bounds__(256) k_group_gemv_simple(const __grid_constant__ GArgs a) {
  const int o = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (o >= a.rows) return;
  float acc[kMaxTokens];
#pragma unroll
  for (int b = 0; b < kMaxTokens; ++b) acc[b] = 0.0f;
  const int bytes = (a.cols + 1) / 2;
  const uint8_t* row = a.codes + static_cast<int64_t>(o) * bytes;
  for (int i = lane; i < bytes; i += 32) {
    const uint32_t two = row[i];
    const int64_t at = static_cast<int64_t>(o) * a.groups + 2 * i / a.group;
    const float s = scale_value(a.scales[at], a.scale_type);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = 2 * i + e;
      if (k >= a.cols) break;
      const uint32_t c = e ? two >> 4 : two & 15u;
      float w;
      if (kCode == kCodeFp4) w = dec_fp4_ref(c);
      else if (kCode == kCodeInt4) w = static_cast<float>(static_cast<int>(c ^ 8u) - 8);
      else w = static_cast<float>(static_cast<int>(c) - static_cast<int>(a.zeros[at]));
      w *= s;
#pragma unroll
      for (int b = 0; b < kMaxTokens; ++b)
        if (b < a.n) acc[b] += w * a.x[b * a.x_ld + k];
    }
  }
#pragma unroll
  for (int b = 0; b < kMaxTokens; ++b) {
    if (b >= a.n) break;
    float v = acc[b];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (lane == 0) g_write(a, o, b, v);
  }
}

// One warp per (row, group): the group's range gives its scale, rounded to the scale's type before
// the codes are chosen, so that decoding multiplies by what the codes were divided by.
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
  for (int k = k0 + lane; k < k1; k += 32) {
    lo = fminf(lo, w[k]);
    hi = fmaxf(hi, w[k]);
  }
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
  for (void* p : {static_cast<void*>(codes), static_cast<void*>(scales), static_cast<void*>(zeros), static_cast<void*>(bias)})
    if (p) cudaFree(p);
}

static Status gdense_fill(GroupDense* g, const GroupDenseSrc& src) {
  WB_CUDA(cudaSetDevice(g->device));
  const size_t n_codes = static_cast<size_t>(g->rows) * ((g->cols + 1) / 2), n_groups = static_cast<size_t>(g->rows) * g->groups;
  const cudaMemcpyKind kind = src.on_device ? cudaMemcpyDeviceToDevice : cudaMemcpyHostToDevice;
  WB_CUDA(cudaMalloc(&g->codes, n_codes));
  WB_CUDA(cudaMemcpy(g->codes, src.codes, n_codes, kind));
  WB_CUDA(cudaMalloc(&g->scales, n_groups * 2));
  WB_CUDA(cudaMemcpy(g->scales, src.scales, n_groups * 2, kind));
  if (g->code == kCodeUint4) {
    WB_CUDA(cudaMalloc(&g->zeros, n_groups));
    WB_CUDA(cudaMemcpy(g->zeros, src.zeros, n_groups, kind));
  }
  g->bias_len = static_cast<int>(src.bias_len < static_cast<size_t>(g->rows) ? src.bias_len : g->rows);
  if (g->bias_len > 0) {
    WB_CUDA(cudaMalloc(&g->bias, static_cast<size_t>(g->bias_len) * 8));
    WB_CUDA(cudaMemcpy(g->bias, src.bias, static_cast<size_t>(g->bias_len) * 8, cudaMemcpyHostToDevice));
  }
  return cuda_status(cudaDeviceSynchronize(), "group dense mount");
}

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
    delete g;
    return st;
  }
  *out = g;
  return Status::Ok();
}

Status gdense_forward(GroupDense* g, int n, const float* x, int64_t x_ld, float* pre, float* post, cudaStream_t st) {
  WB_CUDA(cudaSetDevice(g->device));
  GArgs a;
  a.codes = g->codes;
  a.scales = g->scales;
  a.zeros = g->zeros;
  a.bias = g->bias;
  a.rows = g->rows;
  a.cols = g->cols;
  a.group = g->group;
  a.groups = g->groups;
  a.scale_type = g->scale_type;
  a.act = g->act;
  a.bias_len = g->bias_len;
  a.x_ld = x_ld;
  for (int b = 0; b < n; b += kMaxTokens) {
    a.n = n - b < kMaxTokens ? n - b : kMaxTokens;
    a.x = x + b * x_ld;
    a.pre = pre ? pre + static_cast<int64_t>(b) * g->rows : nullptr;
    a.post = post + static_cast<int64_t>(b) * g->rows;
    const int blocks = (g->rows + 7) / 8;
    if (g->code == kCodeFp4) k_group_gemv_simple<kCodeFp4><<<blocks, 256, 0, st>>>(a);
    else if (g->code == kCodeInt4) k_group_gemv_simple<kCodeInt4><<<blocks, 256, 0, st>>>(a);
    else k_group_gemv_simple<kCodeUint4><<<blocks, 256, 0, st>>>(a);
    WB_TRY(cuda_status(cudaGetLastError(), "group gemv launch"));
  }
  return Status::Ok();
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
