// Distillation from a teacher's top logits on the student's (padded, 16-bit or float32) logits, forward and backward: the soft-target
// counterpart of the cross entropy in xent.cu, on the same logits.  With q = softmax(v / T) over the teacher's k entries (v_i, idx_i) of a
// row and z the student's logits,
//     loss[r]   = T^2 sum_i q_i (log q_i - (z[r, idx_i] / T - lse[r])),      lse[r] = log sum_j exp(z[r, j] / T)
//     dz[r, j]  = T (exp(z[r, j] / T - lse[r]) - sum_{i: idx_i = j} q_i) * g     (0 in rows without a teacher and in padded columns)
// The teacher's tail is not modelled: its top entries are renormalised.  Both passes are bound by HBM: one read of the logits forward, one
// read and one write backward (8192 x 50304 bf16: 129 us with 16 teacher entries and 137 with 32 = 6.4 and 6.0 TB/s, and 266 us = 6.2 TB/s, of 6.5
// for a copy); q is kept (k numbers per row), the logits' log-probabilities are not.
//
// lse = M / T + log S (M the row's largest logit, S the sum of exp((z - M) / T)) loses log S where M / T is large: at 1e4 a tenth of a percent of
// every probability, and all of it in a row of nothing but the type's lowest value.  So it is kept as two floats, lse[r] rounded and what that
// rounding left out: live_rows[r] is 0 in rows without a teacher and the bits of that rest in the others (-0 for none).  The backward pass takes
// differences from a logit near T lse and adds what that one is off, in both floats.  From |lse| = 2^24 on M / T alone fills both (or is beyond
// float32): there the rest is log S, and the backward pass finds M again.
#include "head_loss.cuh"
#include "tcgen05.cuh"

#include <cfloat>

namespace lancet {
namespace head {

constexpr float kLseTwoFloats = 0x1p24f;   // below it the two floats hold log-sum-exp to 2^-24 of 1 + log S

constexpr int kMeanThreads = 1024;
__global__ void __launch_bounds__(kMeanThreads)
mean_kernel(const float* __restrict__ loss_rows, const int32_t* __restrict__ live_rows, int rows, float* __restrict__ mean,
            float* __restrict__ inv_live) {
  chain_enter();
  __shared__ double s_sum[kMeanThreads / 32];
  __shared__ int s_live[kMeanThreads / 32];
  double sum = 0.0;
  int live = 0;
  for (int r = threadIdx.x; r < rows; r += kMeanThreads) {
    sum += (double)loss_rows[r];
    live += live_rows[r] != 0;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    live += __shfl_xor_sync(0xffffffffu, live, d);
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_live[threadIdx.x >> 5] = live;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    int n = 0;
    for (int w = 0; w < kMeanThreads / 32; ++w) {
      total += s_sum[w];
      n += s_live[w];
    }
    n = n > 1 ? n : 1;
    *mean = (float)(total / n);
    *inv_live = 1.0f / (float)n;
  }
}

int launch_mean(const float* loss_rows, const int32_t* live_rows, int rows, float* mean, float* inv_live, cudaStream_t st) {
  launch_chained(mean_kernel, dim3(1), dim3(kMeanThreads), 0, st, loss_rows, live_rows, rows, mean, inv_live);
  return launch_status("mean_kernel");
}

using gemm::add2;
using gemm::f32x2;
using gemm::mul2;
using gemm::pack2;
using gemm::splat2;
using gemm::unpack2;

template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// Elements of a row before the first 16-byte boundary (the whole row where T's own alignment is all there is to have).
template <typename T>
__device__ __forceinline__ int row_head(const T* row, int n) {
  const int head = (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T));
  return head < n ? head : n;
}

// Running maximum m (of the raw values, so that masks of the type's lowest value stay finite) and sum s of 2^((x - m) c).  m starts at
// the lowest finite float: a value of -inf then adds 0, and a row of nothing but -inf ends with s = 0.
__device__ __forceinline__ void add_one(float& m, float& s, float x, float c) {
  if (x > m) {
    s = s * ex2f((m - x) * c) + 1.0f;
    m = x;
  } else {
    s += ex2f((x - m) * c);
  }
}
// Largest value of a 16-byte vector: 16-bit types are compared in pairs.
__device__ __forceinline__ float vec_max(const Vec<float>& a) { return fmaxf(fmaxf(a.v[0], a.v[1]), fmaxf(a.v[2], a.v[3])); }
__device__ __forceinline__ float vec_max(const Vec<__half>& a) {
  const __half2* p = reinterpret_cast<const __half2*>(a.v);
  const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(const Vec<__nv_bfloat16>& a) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(a.v);
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
template <typename T>
__device__ __forceinline__ void add_vec(float& m, float& s, const Vec<T>& a, float c) {
  constexpr int N = Vec<T>::N;
  const float vm = vec_max(a);
  if (vm > m) {
    s *= ex2f((m - vm) * c);
    m = vm;
  }
  const f32x2 mm = splat2(-m), cc = splat2(c);   // two values per instruction, difference before the scale
  f32x2 sum = 0ull;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    float x, y;
    unpack2(mul2(add2(pack2(Num<T>::to_f(a.v[j]), Num<T>::to_f(a.v[j + 1])), mm), cc), x, y);
    sum = add2(sum, pack2(ex2f(x), ex2f(y)));
  }
  float x, y;
  unpack2(sum, x, y);
  s += x + y;
}
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float c) {
  const float mm = fmaxf(m, m2);
  s = s * ex2f((m - mm) * c) + s2 * ex2f((m2 - mm) * c);
  m = mm;
}

// Threads of a row's block.  A block has fixed steps at both ends (the teacher's softmax, the joins, a last round of loads that does not fill the
// block), so smaller blocks with more rows under way read faster; the backward pass, which has no such steps, writes long rows faster
// from large blocks.  8192 x 50304 bf16, 256 / 128 / 64 threads: forward 143 / 132 / 137 us, backward 268 / 276 / 287; 60000 x 4500: forward
// 338 / 191 / 163, backward 305 / 212 / 183.
constexpr int SHORT_ROW_BYTES = 16384, SHORT_THREADS = 64, FWD_THREADS = 128, BWD_THREADS = 256;

// A row is read by one block, or with few rows by the blocks of a cluster: contiguous shares of its 16-byte vectors, the maxima and sums
// joined through the cluster's shared memory in rank order.
struct Share {
  int v0, v1;         // vectors of this block
  bool first, last;   // has the elements before the first vector, behind the last one
};
__device__ __forceinline__ Share share_of(int nv, int part, int parts) {
  Share s;
  s.v0 = (int)((long long)nv * part / parts);
  s.v1 = (int)((long long)nv * (part + 1) / parts);
  s.first = part == 0;
  s.last = part == parts - 1;
  return s;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_load(const float* p, int rank) {
  uint32_t local = (uint32_t)__cvta_generic_to_shared(p), remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads)
distill_fwd_kernel(const T* __restrict__ x, long long ld, const void* __restrict__ values, int vdtype, const long long* __restrict__ indices,
                   int k, float inv_t, int V, int parts, float* __restrict__ loss, float* __restrict__ lse, float* __restrict__ weights,
                   int32_t* __restrict__ live_rows) {
  chain_enter();
  constexpr int N = Vec<T>::N;
  __shared__ float s_q[kMaxTop];
  __shared__ int s_idx[kMaxTop];
  __shared__ float s_m[kThreads / 32], s_s[kThreads / 32];
  __shared__ float s_part[2];
  __shared__ int s_live;
  const int part = blockIdx.x % parts;   // rank in the row's cluster
  const long long r = blockIdx.x / parts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float c = inv_t * kLog2e;
  if (warp == 0) {
    const bool live = teacher_row(values, vdtype, indices, r, k, inv_t, V, s_q, s_idx);
    if (lane == 0) s_live = live;
  }
  __syncthreads();
  if (part == 0)
    for (int i = threadIdx.x; i < k; i += kThreads) weights[r * k + i] = class_weight(s_q, s_idx, k, i);
  if (!s_live) {   // in all blocks of the cluster alike
    if (part == 0 && threadIdx.x == 0) {
      loss[r] = 0.f;
      lse[r] = 0.f;
      live_rows[r] = 0;
    }
    return;
  }
  const T* row = x + r * ld;
  float m = -FLT_MAX, s = 0.f;
  const int head = row_head(row, V);
  const int nv = (V - head) / N;
  const Share sh = share_of(nv, part, parts);
  auto get = [&](int v) {   // each value is read once
    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(row + head) + v);
    return *reinterpret_cast<const Vec<T>*>(&q);
  };
  if (sh.first && (int)threadIdx.x < head) add_one(m, s, Num<T>::to_f(row[threadIdx.x]), c);
  int i = sh.v0 + threadIdx.x;
  for (; i + 3 * kThreads < sh.v1; i += 4 * kThreads) {   // four loads in flight
    const Vec<T> a = get(i), b = get(i + kThreads), d = get(i + 2 * kThreads), e = get(i + 3 * kThreads);
    add_vec(m, s, a, c);
    add_vec(m, s, b, c);
    add_vec(m, s, d, c);
    add_vec(m, s, e, c);
  }
  for (; i < sh.v1; i += kThreads) add_vec(m, s, get(i), c);
  if (sh.last)
    for (int j = head + nv * N + threadIdx.x; j < V; j += kThreads) add_one(m, s, Num<T>::to_f(row[j]), c);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, d), s2 = __shfl_xor_sync(0xffffffffu, s, d);
    merge(m, s, m2, s2, c);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_s[warp] = s;
  }
  __syncthreads();
  float M = s_m[0], S = s_s[0];
  for (int w = 1; w < kThreads / 32; ++w) merge(M, S, s_m[w], s_s[w], c);
  if (parts > 1) {
    if (threadIdx.x == 0) {
      s_part[0] = M;
      s_part[1] = S;
    }
    __syncwarp();
    cluster_barrier();
    if (part == 0 && warp == 0)
      for (int p = 1; p < parts; ++p) merge(M, S, cluster_load(&s_part[0], p), cluster_load(&s_part[1], p), c);
    cluster_barrier();   // no block leaves while its sums are read
  }
  if (part == 0 && warp == 0) {
    const float log_s = logf(S);
    const float l = fmaf(M, inv_t, log_s);
    const float rest = fabsf(l) >= kLseTwoFloats ? log_s : fmaf(M, inv_t, -l) + log_s;
    float sum = 0.f;
    for (int e = lane; e < k; e += 32)
      if (s_q[e] != 0.f) sum += s_q[e] * (logf(s_q[e]) - ((Num<T>::to_f(row[s_idx[e]]) - M) * inv_t - log_s));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) {
      lse[r] = l;
      loss[r] = sum / (inv_t * inv_t);
      live_rows[r] = rest == 0.f ? (int32_t)0x80000000 : __float_as_int(rest);
    }
  }
}

// Largest value of a row, in all threads of its block.  A call, so that the rows that need it cost the others no registers.
template <typename T, int kThreads>
__device__ __noinline__ float block_max(const T* row, int V) {
  __shared__ float s_m[kThreads / 32];
  float m = -INFINITY;
#pragma unroll 1
  for (int j = threadIdx.x; j < V; j += kThreads) m = fmaxf(m, Num<T>::to_f(row[j]));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, s_m[w]);
  return m;
}

// 32 registers a thread: whole SMs of threads.  With the 42 that the compiler takes unbounded (6 blocks of 256 per SM) 8192 x 50304 bf16 ran 259 us
// for 267, but 500 x 50257 20.0 for 16.8 and 60000 x 4500 187 for 177.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == BWD_THREADS ? 8 : 28)
distill_bwd_kernel(const T* __restrict__ x, long long ld, const long long* __restrict__ indices, const float* __restrict__ weights,
                   const int32_t* __restrict__ live_rows, int k, float inv_t, int V, int cols, int parts, const float* __restrict__ lse,
                   const float* __restrict__ gout, const float* __restrict__ inv_live, float scale, T* __restrict__ dx, long long ldd) {
  chain_enter();
  constexpr int N = Vec<T>::N;
  const int part = blockIdx.x % parts;
  const long long r = blockIdx.x / parts;
  const T* row = x + r * ld;
  T* drow = dx + r * ldd;
  const int rest = live_rows[r];
  const bool live = rest != 0;
  const float g = scale * (gout ? *gout : 1.f) * (inv_live ? *inv_live : 1.f) / inv_t;
  const float c = inv_t * kLog2e, l = lse[r];
  float base = l / inv_t, off = __int_as_float(rest) - fmaf(base, inv_t, -l);   // log-sum-exp = base / T + off
  if (live && fabsf(l) >= kLseTwoFloats) {   // the same in all threads
    base = block_max<T, kThreads>(row, V);
    off = __int_as_float(rest);
  }
  const float part_g = ex2f(-off * kLog2e) * g;   // off goes into the factor of the gradient
  // Vectors where both rows meet 16-byte boundaries at the same element; the blocks of a row take contiguous shares of them.  Elsewhere (columns
  // sliced off a padded matrix) single elements: 8192 x 50257 of 50304 bf16 774 us for 266 with the padding named by V, float32 835 for 522.
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(drow)) & 15) == 0;
  const int head = same ? row_head(row, V) : 0;
  const int nv = same ? (V - head) / N : 0;
  const Share sh = share_of(nv, part, parts);
  const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + head);
  Vec<T>* dv = reinterpret_cast<Vec<T>*>(drow + head);
  auto grad = [&](float v) { return Num<T>::from_f(ex2f((v - base) * c) * part_g); };   // differences of raw values, as in the forward pass
  auto grad_vec = [&](const Vec<T>& v) {
    Vec<T> o;
    const f32x2 bb = splat2(-base), cc = splat2(c), gg = splat2(part_g);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float x, y;
      unpack2(mul2(add2(pack2(Num<T>::to_f(v.v[j]), Num<T>::to_f(v.v[j + 1])), bb), cc), x, y);
      unpack2(mul2(pack2(ex2f(x), ex2f(y)), gg), x, y);
      o.v[j] = Num<T>::from_f(x);
      o.v[j + 1] = Num<T>::from_f(y);
    }
    return o;
  };
  // single elements: those outside the vectors, or without vectors this block's share of the row
  const int tail0 = head + nv * N;
  const Share single = share_of(cols - tail0, same ? 0 : part, same ? 1 : parts);
  auto one = [&](int j) { drow[j] = live && j < V ? grad(Num<T>::to_f(row[j])) : Num<T>::from_f(0.f); };
  if (sh.first && (int)threadIdx.x < head) one(threadIdx.x);
  if (sh.last || !same)
    for (int j = tail0 + single.v0 + threadIdx.x; j < tail0 + single.v1; j += kThreads) one(j);
  if (!live) {
    Vec<T> z;
#pragma unroll
    for (int j = 0; j < N; ++j) z.v[j] = Num<T>::from_f(0.f);
    for (int i = sh.v0 + threadIdx.x; i < sh.v1; i += kThreads) dv[i] = z;
    return;
  }
  int i = sh.v0 + threadIdx.x;
  for (; i + 3 * kThreads < sh.v1; i += 4 * kThreads) {
    const Vec<T> a0 = rv[i], a1 = rv[i + kThreads], a2 = rv[i + 2 * kThreads], a3 = rv[i + 3 * kThreads];
    dv[i] = grad_vec(a0);
    dv[i + kThreads] = grad_vec(a1);
    dv[i + 2 * kThreads] = grad_vec(a2);
    dv[i + 3 * kThreads] = grad_vec(a3);
  }
  for (; i < sh.v1; i += kThreads) dv[i] = grad_vec(rv[i]);
  __syncthreads();
  // the teacher's classes, each by the block that wrote its element: difference in float32, rounded once (entries of one class write the same
  // value)
  const int from = same ? (sh.first ? 0 : head + sh.v0 * N) : single.v0;
  const int to = same ? (sh.last ? V : head + sh.v1 * N) : single.v1;
  for (int e = threadIdx.x; e < k; e += kThreads) {
    const long long at = indices[r * k + e];
    if (at >= from && at < to && at < V) drow[at] = Num<T>::from_f(ex2f((Num<T>::to_f(row[at]) - base) * c) * part_g - weights[r * k + e] * g);
  }
}

static bool short_rows(int vocab, int bytes) { return (long long)vocab * bytes < SHORT_ROW_BYTES; }
// Blocks per row: several while there are no more than 4 (forward; 8 backward) blocks per SM and each has 16 KB of the row.  50257 bf16, one /
// several blocks: 7 rows forward 12.7 / 10.6 us, backward 8.4 / 6.3; 500 rows forward 18.8 / 21.0 (so one), backward 18.3 / 16.7.
constexpr int FWD_BLOCKS_PER_SM = 4, BWD_BLOCKS_PER_SM = 8;
static int parts_for(int rows, int vocab, int bytes, int blocks_per_sm) {
  int parts = 1;
  while (parts < 8 && 2ll * parts * rows <= (long long)blocks_per_sm * sm_count() && (long long)vocab * bytes / (2 * parts) >= 16384) parts *= 2;
  return parts;
}

// A chained launch, in clusters of `parts` blocks where the kernel joins its blocks' sums.
template <typename... KArgs, typename... Args>
static int launch_rows(void (*kernel)(KArgs...), const char* name, int rows, int parts, int threads, bool cluster, cudaStream_t st,
                       Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * parts);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = chained_launch_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster && parts > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  return launch_status(name);
}

template <typename T>
static int fwd_t(const void* x, long long ld, const void* values, int vdtype, const long long* indices, int k, float inv_t, int rows, int vocab,
                 float* loss, float* lse, float* weights, int32_t* live_rows, cudaStream_t st) {
  const bool few = short_rows(vocab, sizeof(T));
  const int threads = few ? SHORT_THREADS : FWD_THREADS, parts = parts_for(rows, vocab, sizeof(T), FWD_BLOCKS_PER_SM);
  return launch_rows(few ? distill_fwd_kernel<T, SHORT_THREADS> : distill_fwd_kernel<T, FWD_THREADS>, "distill_fwd_kernel", rows, parts, threads,
                     true, st, static_cast<const T*>(x), ld, values, vdtype, indices, k, inv_t, vocab, parts, loss, lse, weights, live_rows);
}

template <typename T>
static int bwd_t(const void* x, long long ld, const long long* indices, const float* weights, const int32_t* live_rows, int k, float inv_t,
                 int rows, int vocab, int cols, const float* lse, const float* gout, const float* inv_live, float scale, void* dx,
                 long long ldd, cudaStream_t st) {
  const bool few = short_rows(vocab, sizeof(T));
  const int threads = few ? SHORT_THREADS : BWD_THREADS, parts = parts_for(rows, vocab, sizeof(T), BWD_BLOCKS_PER_SM);
  return launch_rows(few ? distill_bwd_kernel<T, SHORT_THREADS> : distill_bwd_kernel<T, BWD_THREADS>, "distill_bwd_kernel", rows, parts, threads,
                     false, st, static_cast<const T*>(x), ld, indices, weights, live_rows, k, inv_t, vocab, cols, parts, lse, gout, inv_live,
                     scale, static_cast<T*>(dx), ldd);
}

}  // namespace head
}  // namespace lancet

extern "C" {
using namespace lancet;

int lancet_distill_fwd(const void* logits, long long ld, const void* top_values, int values_dtype, const long long* top_indices, int k,
                       float temperature, int rows, int vocab, int dtype, float* loss_rows, float* lse_rows, float* class_weights,
                       int32_t* live_rows, float* mean, float* inv_live, lancet_stream_t stream) {
  LANCET_REQUIRE(rows >= 0 && rows <= head::kMostSize && vocab >= 1 && vocab <= head::kMostSize && ld >= vocab && valid_dtype(dtype) &&
                     valid_dtype(values_dtype), LANCET_ERR_INVALID,
                 "lancet_distill_fwd: bad rows=%d, vocab=%d, row stride %lld or dtype", rows, vocab, ld);
  LANCET_REQUIRE(k >= 1 && k <= head::kMaxTop, LANCET_ERR_INVALID, "lancet_distill_fwd: k=%d top entries (1 to %d)", k, head::kMaxTop);
  LANCET_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, LANCET_ERR_INVALID, "lancet_distill_fwd: temperature %g outside [0.001, 1000]",
                 (double)temperature);
  LANCET_REQUIRE(mean && inv_live && (rows == 0 || (logits && top_values && top_indices && loss_rows && lse_rows && class_weights && live_rows)),
                 LANCET_ERR_NULL, "lancet_distill_fwd: null pointer argument");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows > 0)
    if (int rc = LANCET_DISPATCH_DTYPE(dtype, head::fwd_t, logits, ld, top_values, values_dtype, top_indices, k, 1.0f / temperature, rows,
                                       vocab, loss_rows, lse_rows, class_weights, live_rows, st))
      return rc;
  return head::launch_mean(loss_rows, live_rows, rows, mean, inv_live, st);
}

int lancet_distill_bwd(const void* logits, long long ld, const long long* top_indices, const float* class_weights, const int32_t* live_rows,
                       int k, float temperature, int rows, int vocab, int cols, int dtype, const float* lse_rows, const float* grad_out,
                       const float* inv_live, float scale, void* dlogits, long long ldd, lancet_stream_t stream) {
  LANCET_REQUIRE(rows >= 0 && rows <= head::kMostSize && vocab >= 1 && cols >= vocab && cols <= head::kMostSize && ld >= vocab && ldd >= cols &&
                     valid_dtype(dtype), LANCET_ERR_INVALID,
                 "lancet_distill_bwd: bad rows=%d, vocab=%d, cols=%d, row strides %lld / %lld or dtype", rows, vocab, cols, ld, ldd);
  LANCET_REQUIRE(k >= 1 && k <= head::kMaxTop, LANCET_ERR_INVALID, "lancet_distill_bwd: k=%d top entries (1 to %d)", k, head::kMaxTop);
  LANCET_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, LANCET_ERR_INVALID, "lancet_distill_bwd: temperature %g outside [0.001, 1000]",
                 (double)temperature);
  if (rows == 0) return LANCET_OK;
  LANCET_REQUIRE(logits && top_indices && class_weights && live_rows && lse_rows && dlogits, LANCET_ERR_NULL,
                 "lancet_distill_bwd: null pointer argument");
  return LANCET_DISPATCH_DTYPE(dtype, head::bwd_t, logits, ld, top_indices, class_weights, live_rows, k, 1.0f / temperature, rows, vocab, cols,
                               lse_rows, grad_out, inv_live, scale, dlogits, ldd, static_cast<cudaStream_t>(stream));
}
}
