// What the head's losses share: the teacher's distribution over its top entries, sums in the base-2 domain, and the mean
// over live rows.  A teacher gives k (value, index) pairs per row.  An entry counts if its index names a class
// (0 <= index < vocab); q = softmax(value / T) over the entries that count.  A row without any, or whose counting values are
// all -inf, has no teacher: it is ignored, like a row without a target.
#pragma once
#include "common.cuh"

namespace lancet {
namespace head {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMostSize = 1 << 30;   // rows or columns: 32-bit counters step past the end by less than as much again
constexpr int kMaxTop = 512;   // entries of a teacher's row: they are held in shared memory

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Teacher distribution of one row by one warp: q[i] and idx[i] (-1: does not count) go to shared memory.  Returns whether the row has a
// teacher.  The differences are taken before the division by T, so that values of the type's lowest magnitude stay exact.
__device__ __forceinline__ bool teacher_row(const void* values, int vdtype, const long long* __restrict__ indices, long long row, int k,
                                            float inv_t, int vocab, float* q, int* idx) {
  const int lane = threadIdx.x & 31;
  float vmax = -INFINITY;
  bool nan = false;
  for (int i = lane; i < k; i += 32) {
    const long long at = indices[row * k + i];
    const bool counts = at >= 0 && at < vocab;
    const float v = counts ? load_as_float(values, vdtype, (size_t)row * k + i) : -INFINITY;
    idx[i] = counts ? (int)at : -1;
    q[i] = v;
    vmax = fmaxf(vmax, v);
    nan |= (v != v);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
  nan = __any_sync(0xffffffffu, nan);
  const bool live = nan || vmax > -INFINITY;
  float sum = 0.f;
  for (int i = lane; i < k; i += 32) {
    const float e = live && idx[i] >= 0 ? expf((q[i] - vmax) * inv_t) : 0.f;
    q[i] = e;
    sum += e;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  for (int i = lane; i < k; i += 32) q[i] = live && idx[i] >= 0 ? q[i] / sum : 0.f;
  __syncwarp();
  return live;
}

// Weight of entry i's class: its own q plus those of other entries that name the same class.
__device__ __forceinline__ float class_weight(const float* q, const int* idx, int k, int i) {
  const int at = idx[i];
  float s = 0.f;
  for (int j = 0; j < k; ++j) s += idx[j] == at ? q[j] : 0.f;
  return s;
}

// mean = sum of the row losses / max(live rows, 1), inv_live = 1 / max(live rows, 1), the live rows counted from per-row flags.  One block,
// fixed order, 64-bit sums.
int launch_mean(const float* loss_rows, const int32_t* live_rows, int rows, float* mean, float* inv_live, cudaStream_t st);

}  // namespace head
}  // namespace lancet
