// gdense.hpp -- a Dense layer of 4-bit codes with one scale (and zero point) per group of inputs.
//
// No counterpart in the reference, whose 4-bit stores carry one scale per tensor
// (src/weights/native_codec.cpp:174-262). y[b][o] = act(sum_g s[o][g] * sum_{i in g} v(c[o][i]) *
// x[b][i] + bias[o]), v(c) the E2M1 value (FP4), the two's complement nibble (Int4) or c - zero[o][g]
// (Uint4). Bias, activation and the float roundings around them are the Dense layer's.
#pragma once

#include "common.hpp"

namespace wb {

constexpr int kCodeInt4 = 14, kCodeUint4 = 15, kCodeFp4 = 16;  // ids of the reference's DType table
constexpr int kScaleF16 = 2, kScaleBF16 = 3;

struct GroupDense {
  int device = 0;
  int rows = 0, cols = 0;  // outputs, inputs
  int group = 0, groups = 0;
  int code = 0, act = -1;
  int scale_type = 0;  // kScaleF16, kScaleBF16, or the kernel's own kind of very large BFloat16 scales
  uint8_t* w = nullptr;  // codes, scales and zero points in the kernel's records (gdense.cu)
  double* bias = nullptr;
  int bias_len = 0;
  int sms = 148;
  uint8_t* work = nullptr;   // the one allocation behind what follows
  int* tickets = nullptr;
  float* part = nullptr;
  float* slab_sum = nullptr;
  ~GroupDense();
};

struct GroupDenseSrc {
  const uint8_t* codes = nullptr;
  const void* scales = nullptr;
  const uint8_t* zeros = nullptr;
  bool on_device = false;
  const double* bias = nullptr;  // host
  size_t bias_len = 0;
};

Status gdense_mount(int device, int rows, int cols, int group, int code, int scale_type, int act, const GroupDenseSrc& src,
                    GroupDense** out);
// x [n][cols] (rows x_ld apart), pre (may be null) and post [n][rows].
Status gdense_forward(GroupDense* g, int n, const float* x, int64_t x_ld, float* pre, float* post, cudaStream_t st);

// The launch plan of a call of n tokens (1..8) on a GPU of `sms` multiprocessors, host arithmetic only:
// slabs, chunks of a slab, blocks of a slab, runs are the warps', runs are whole row groups, bytes of
// shared memory, row groups, chunks, runs of a slab, row groups that runs cut. Returns their number.
int gdense_plan_values(int rows, int cols, int group, int code, int sms, int n, int64_t* out, int count);

// W [rows][cols] float32 -> codes, scales, zeros (Uint4) in the layout gdense_mount takes.
Status group_quantize(int rows, int cols, int group, int code, int scale_type, const float* W, uint8_t* codes, void* scales,
                      uint8_t* zeros, cudaStream_t st);

} // namespace wb
