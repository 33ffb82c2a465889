// Losses of the language-model head from its hidden rows, without keeping the logits: cross entropy against target tokens and distillation
// from a teacher's top logits, forward and backward.  With h [rows][width], W [classes][width] and z = h W^T (never in memory),
//     lse[r]  = log sum_j exp(z[r, j] / T)                         (T = 1 for the cross entropy)
//     loss[r] = lse[r] - z[r, t_r]          or   T^2 sum_i q_i (log q_i - (z[r, idx_i] / T - lse[r])),   q = softmax(v / T)
//     dz[r, j] = T (exp(z[r, j] / T - lse[r]) - sum_{i: idx_i = j} q_i) g,     dh = dz W,     dW = dz^T h      (one entry with q = 1 for a target)
// The forward pass is one product whose epilogue reduces each tile's columns to a maximum and a sum per row, and a kernel that joins them and
// adds the logits at the targets.  The backward pass walks the vocabulary in pieces of up to 1 GiB of dz (8192 x 50257: all of it in one piece): the
// same product again, with an epilogue that writes exp(z / T - lse) in 16 bits (less 1 at a target; a teacher's k differences are placed by a
// small kernel), and two products from that piece.  2 + 2 + 4 flops per row, class and width element, against 2 + 4 with the logits kept.
//
// Roundings: dz goes to the tensor cores in the operands' 16 bits, the one rounding beside the results' own, where a loss on 16-bit logits rounds its
// gradient too; products of a float32 dz would take several 16-bit products or tf32's half rate.  Distance of dh and dW from the definition at
// 8192 x 50257 x 1024 bf16: 1.9e-3 and 2.0e-3 relative, 1.7e-3 with a float32 dz, 3.0e-3 with 16-bit logits kept.  z is what the tensor cores sum,
// which they cut short (see finish_rows_kernel), and enters exp2 by one fused multiply-add, so a probability carries some 2^-23 |z| / T.  Log-sum-exp is
// one float32: its rounding of 2^-24 |lse| is below that.
//
// Rows without a target (or teacher) take no part: the first kernel of each pass packs the live rows together, every product works on their
// number, which stays on the device, and the gradient rows go back through the row list.  So an ignored row may hold anything, NaN
// included, and costs a copy's time only.
//
// All products run on one kernel: tcgen05.mma on 256 x 256 tiles of a CTA pair (128 x 256 of one CTA up to 128 rows), operands in
// 128-byte-swizzled tiles staged by TMA, float32 accumulators in TMEM, two of them so that the epilogue of one tile runs under the next
// tile's products; results leave through shared memory as TMA boxes.  Bound by the tensor cores from a few hundred rows on: at 8192 x 50257 x
// 1024 bf16 the four products take 533 (sums), 557 (dz), 559 (dh) and 540 us (dW) alone = 1.51 to 1.58 PFLOP/s, 0.94 to 0.99 of the measured
// burst of a library product; in a loop the power limit holds the step to 2.65 ms (1.27 PFLOP/s, 0.93 of the sustained figure).  With a few
// rows the weight's bytes bound it (read three times, its gradient written once), below about 100 us the host does.
#include "head_loss.cuh"
#include "tcgen05.cuh"

namespace lancet {
namespace head {

using namespace lancet::gemm;

constexpr int BM = 128, BN = 256, BK = 64, UMMA_K = 16;
constexpr int A_STAGE_BYTES = BM * BK * 2;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int TMEM_COLS = 512;
constexpr int ROW_PAD = 256;                    // row buffers hold a multiple of this: whole tiles, in the paired form too
constexpr long long BAND_BYTES = 20ll << 20;    // rows of A swept against all columns before the next band: they stay in L2

// Products (A's and B's rows are M and N):
//   FORM_Z   z tile  = h W^T       M = live rows, N = classes, reduction over the width;    both operands K-major
//   FORM_DH  dh tile = dz W        M = live rows, N = width, reduction over the classes;    W is MN-major
//   FORM_DW  dW tile = dz^T h      M = classes, N = width, reduction over the live rows;    both MN-major
constexpr int FORM_Z = 0, FORM_DH = 1, FORM_DW = 2;
constexpr int EPI_LSE = 0, EPI_PROB = 1, EPI_OUT = 2;

// Boxes of 16-bit results on their way out, 32 rows x 64 columns in the 128-byte swizzle: two per epilogue warp where whole tiles leave this way
// (one is filled while the other leaves), none for the row sums.  The operand stages take what is left of the shared memory.
constexpr int OUT_ROWS = 32, OUT_COLS = BK, OUT_BOX_BYTES = OUT_ROWS * OUT_COLS * 2;
constexpr int SMEM_MOST = 227 * 1024, SMEM_SLACK = 1024 /*alignment*/ + 256 /*barriers*/;
template <int FORM, int EPI, bool CTA2>
struct Cfg {
  static constexpr int OUT_BYTES = EPI_WARPS * OUT_BOX_BYTES * (EPI == EPI_LSE ? 0 : FORM == FORM_DH ? 1 : 2);
  static constexpr int B_COLS = CTA2 ? BN / 2 : BN;
  static constexpr int B_STAGE_BYTES = B_COLS * BK * 2;
  static constexpr int STAGE_BYTES = A_STAGE_BYTES + B_STAGE_BYTES;
  static constexpr int FIT = (SMEM_MOST - SMEM_SLACK - OUT_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;
  static constexpr int SMEM_DATA = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = SMEM_DATA + OUT_BYTES + SMEM_SLACK;
};

struct Params {
  const int32_t* count;   // live rows
  int classes;            // of this piece
  int class0;             // first class of the piece
  int width;
  int* status;
  float c;                // log2(e) / T
  // EPI_LSE: per (column half tile, row) maximum and sum in the base-2 domain
  float2* part;
  long long part_ld;
  const int32_t* tgt;     // target (or the teacher's first class) of every packed row; EPI_LSE: its logit goes to zt; EPI_PROB: or null
  float* zt;
  // EPI_PROB: 2^(z c - lse2[row] + shift) of the piece to tmOut, at the rows' targets (tgt) tdiff[row] instead
  const float* lse2;
  const float* tdiff;
  float shift;
  // EPI_OUT
  void* out;
  int boxes;                // whole rows of the output go out through tmOut (rows on 16-byte boundaries, no row_map)
  const int32_t* row_map;   // output row of packed row i, or null
  const float* grad_out;
  const float* inv_live;
  float scale;
  float* acc;               // float32 sums over the pieces, or null
  long long acc_ld;
  int acc_in, acc_out;      // add the sums so far / store sums instead of the output
  float* slots;             // partial sums of split tiles
};

struct Dims {
  int m, n, k;      // k: length of the reduction
  int mu, nt, kb;   // units of rows (a tile, or a pair's two), column tiles, blocks of the reduction
};
template <int FORM, bool CTA2>
__device__ __forceinline__ Dims dims_of(const Params& p) {
  Dims d;
  const int rows = *p.count;
  d.m = FORM == FORM_DW ? p.classes : rows;
  d.n = FORM == FORM_Z ? p.classes : p.width;
  d.k = FORM == FORM_Z ? p.width : (FORM == FORM_DH ? p.classes : rows);
  const int unit = CTA2 ? 2 * BM : BM;
  d.mu = (d.m + unit - 1) / unit;
  d.nt = (d.n + BN - 1) / BN;
  d.kb = (d.k + BK - 1) / BK;
  return d;
}

// A reduction over classes or rows is long where the tiles are few.  The workers first take whole tiles in turn as long as each gets one;
// what is left (`rem` tiles) is cut along the reduction into equal contiguous ranges, a range per worker, so that all of them end together.
// A range spans two tiles at most; parts of a tile go to float32 slots (2 per worker) and are added in order by join_tiles_kernel.
// Cutting pays when the idle share of the last turn, (workers - rem) / workers x kb blocks of 512 clocks, costs more than the parts' way through
// memory and their sum: from 32 blocks on for a few tiles, whose parts stay small, and from 56 on for more (the sides meet between 50 and 62
// blocks).  Captured passes of one gradient, whole tiles / cut, us: few: dW of 2500 rows, 1 tile, 39 blocks 25.9 / 23.0; dh of 300 x 2500 x 768,
// 6 tiles, 37 blocks 29.2 / 28.4, at 2000 classes, 29 blocks 26.9 / 27.9.  More: dW of 3000 x 2000 x 512, 16 tiles, 37 blocks 35.3 / 41.5, of 5000
// rows, 62 blocks 49.0 / 48.3; dh of 2264 x 3500 x 256, 9 tiles, 48 blocks 37.6 / 39.2; of 8152 x 6000 x 256, 32 tiles, 53 blocks 82.0 / 79.2; of
// 100 x 4300 x 7680, 30 tiles, 54 blocks 95.6 / 102.5.  And it pays when that share is more than a
// quarter of all turns: below that the GPU, which runs long products at its power limit, clocks higher while some SMs idle (8192 x 50257 x 1024,
// 128 tiles on 74 pairs: 2.67 / 2.77 ms in a loop).
constexpr int SPLIT_MIN_KB = 32, SPLIT_MIN_KB_MANY = 56;
constexpr int SPLIT_FEW = 12;   // few: as many workers for each tile
constexpr int SPLIT_MIN_PART = 4;
struct Split {
  int full, rem, parts, kb;   // whole tiles, tiles that are cut, ranges they are cut into, blocks of a tile
  long long iters;
  __host__ __device__ long long begin(int w) const { return iters * w / parts; }
};
__host__ __device__ __forceinline__ Split split_of(int n_tiles, int kb, int workers) {
  Split s = {n_tiles, 0, 1, kb, 0};
  const int rem = n_tiles % workers;
  const long long idle = workers - rem, turns = (n_tiles + workers - 1) / workers;
  const long long min_kb = workers >= SPLIT_FEW * rem ? SPLIT_MIN_KB : SPLIT_MIN_KB_MANY;
  if (rem > 0 && idle * kb > min_kb * workers && 4 * idle > turns * workers) {
    s.full = n_tiles - rem;
    s.rem = rem;
    s.iters = (long long)rem * kb;
    long long parts = s.iters / SPLIT_MIN_PART;
    parts = parts < rem ? rem : parts;
    s.parts = (int)(parts > workers ? workers : parts);
  }
  return s;
}
// The items of one worker: a tile, the blocks [k0, k1) of its reduction, and the slot of a partial sum (-1: the whole tile).
struct Walk {
  Split s;
  int worker, workers, next;
  long long pos, end, first;
  int t, k0, k1, slot;
  __device__ __forceinline__ Walk(int n_tiles, int kb, int w, int n, bool may_split) : worker(w), workers(n), next(w) {
    s = may_split ? split_of(n_tiles, kb, n) : Split{n_tiles, 0, 1, kb, 0};
    pos = end = first = 0;
    if (s.rem > 0 && w < s.parts) {
      first = pos = s.begin(w);
      end = s.begin(w + 1);
    }
  }
  __device__ __forceinline__ bool step() {
    if (next < s.full) {
      t = next;
      next += workers;
      k0 = 0;
      k1 = s.kb;
      slot = -1;
      return true;
    }
    if (pos >= end) return false;
    const int j = (int)(pos / s.kb);
    k0 = (int)(pos - (long long)j * s.kb);
    k1 = (int)min((long long)s.kb, k0 + end - pos);
    t = s.full + j;
    slot = k0 == 0 && k1 == s.kb ? -1 : 2 * worker + (pos == first ? 0 : 1);
    pos += k1 - k0;
    return true;
  }
};

struct Tile {
  int mt, nt;   // this CTA's 128-row tile, column tile
};
// FORM_Z: bands of row units that stay in L2, swept against the column tiles.  Otherwise the index with fewer tiles runs fastest: the tiles
// in flight form a block as square as possible and share the most operand slabs.
template <int FORM, bool CTA2>
__device__ __forceinline__ void decode_unit(const Params& p, const Dims& d, int t, int& mu, int& nt) {
  if (FORM == FORM_Z) {
    const long long unit_bytes = (long long)(CTA2 ? 2 * BM : BM) * p.width * 2;
    int band = (int)(BAND_BYTES / unit_bytes);
    band = min(band < 2 ? 2 : band, d.mu);
    const int b = t / (band * d.nt);
    const int in_band = min(band, d.mu - b * band);
    const int r = t - b * band * d.nt;
    nt = r / in_band;
    mu = b * band + (r - nt * in_band);
  } else if (d.nt < d.mu) {
    mu = t / d.nt;
    nt = t - mu * d.nt;
  } else {
    nt = t / d.mu;
    mu = t - nt * d.mu;
  }
}
template <int FORM, bool CTA2>
__device__ __forceinline__ Tile decode(const Params& p, const Dims& d, int t, int rank) {
  int mu, nt;
  decode_unit<FORM, CTA2>(p, d, t, mu, nt);
  Tile tl;
  tl.mt = CTA2 ? 2 * mu + rank : mu;
  tl.nt = nt;
  return tl;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// ACC (EPI_OUT): sums over the pieces pass through p.acc
template <typename T, int FORM, int EPI, bool CTA2, bool ACC>
__global__ void __launch_bounds__(THREADS, 1)
head_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmOut,
                    Params p) {
  using C = Cfg<FORM, EPI, CTA2>;
  constexpr int STAGES = C::STAGES;
  constexpr bool A_MN = FORM == FORM_DW, B_MN = FORM != FORM_Z;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sA = smem;
  unsigned char* sB = smem + STAGES * A_STAGE_BYTES;
  unsigned char* sOut = smem + C::SMEM_DATA;   // the epilogue warps' boxes
  uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + C::OUT_BYTES);
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + STAGES);
  const uint32_t bar_tfull = smem_u32(bars + 2 * STAGES), bar_tempty = smem_u32(bars + 2 * STAGES + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTA2 ? (int)cluster_ctarank() : 0;
  const int worker = CTA2 ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int n_workers = CTA2 ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, CTA2 ? 2 * EPI_WARPS : EPI_WARPS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Earlier kernels' results are read from here on.  TMEM is taken after this wait: a CTA that held it while it waited could keep it from a
  // kernel that it waits for.
  chain_enter();
  if (warp == 1) {
    if (CTA2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CTA2) cluster_sync_all();   // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const Dims d = dims_of<FORM, CTA2>(p);
  Walk walk(d.mu * d.nt, d.kb, worker, n_workers, EPI == EPI_OUT);

  if (warp == 0) {
    // ---------------- TMA producer (one per CTA; in the paired form each CTA loads its own halves) ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const int b_off = CTA2 ? rank * (BN / 2) : 0;   // this CTA's share of the tile's columns
      while (ok && walk.step()) {
        const Tile tl = decode<FORM, CTA2>(p, d, walk.t, rank);
        const int m0 = tl.mt * BM, n0 = tl.nt * BN + b_off;
        for (int kb = walk.k0; kb < walk.k1; ++kb) {
          if (!(ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status, 11))) break;
          const uint32_t a_dst = smem_u32(sA + stage * A_STAGE_BYTES), b_dst = smem_u32(sB + stage * C::B_STAGE_BYTES);
          uint32_t full = bar_full + 8 * stage;
          if (rank == 0) mbar_expect_tx(full, (CTA2 ? 2 : 1) * C::STAGE_BYTES);   // of a pair: both CTAs' bytes
          if (CTA2) full = cluster_addr(full, 0);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if (CTA2) tma_load_2d_pair(dst, map, full, x, y); else tma_load_2d(dst, map, full, x, y);
          };
          if (!A_MN) {
            load(a_dst, &tmA, kb * BK, m0);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) load(a_dst + j * BOX_BYTES, &tmA, m0 + j * 64, kb * BK);
          }
          if (!B_MN) {
            load(b_dst, &tmB, kb * BK, p.class0 + n0);
          } else {
            const int y = (FORM == FORM_DH ? p.class0 : 0) + kb * BK;
#pragma unroll
            for (int j = 0; j < C::B_COLS / 64; ++j) load(b_dst + j * BOX_BYTES, &tmB, n0 + j * 64, y);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (paired form: the even CTA only) ----------------
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = instr_desc<T>(A_MN, B_MN, CTA2 ? 2 * BM : BM, BN);
      int stage = 0;
      uint32_t phase = 0;
      int buf = 0;
      uint32_t tphase = 0;
      bool ok = true;
      while (ok && walk.step()) {
        if (!(ok = mbar_wait(bar_tempty + 8 * buf, ((tphase >> buf) & 1) ^ 1, abort_flag, p.status, 12))) break;
        tc_fence_after();
        const uint32_t tmem_d = tmem_base + (uint32_t)(buf * BN);
        for (int kb = walk.k0; kb < walk.k1; ++kb) {
          if (!(ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, 13))) break;
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + stage * A_STAGE_BYTES);
          const uint32_t b_addr = smem_u32(sB + stage * C::B_STAGE_BYTES);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t adesc = A_MN ? smem_desc_mn_sw128(a_addr + k * 2048) : smem_desc_k_sw128(a_addr + k * UMMA_K * 2);
            const uint64_t bdesc = B_MN ? smem_desc_mn_sw128(b_addr + k * 2048) : smem_desc_k_sw128(b_addr + k * UMMA_K * 2);
            if (CTA2)
              umma_f16_pair(tmem_d, adesc, bdesc, idesc, (kb > walk.k0 || k) ? 1u : 0u);
            else
              umma_f16(tmem_d, adesc, bdesc, idesc, (kb > walk.k0 || k) ? 1u : 0u);
          }
          if (CTA2) umma_commit_pair(bar_empty + 8 * stage); else umma_commit(bar_empty + 8 * stage);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (CTA2) umma_commit_pair(bar_tfull + 8 * buf); else umma_commit(bar_tfull + 8 * buf);
        tphase ^= 1u << buf;
        buf ^= 1;
      }
    }
  } else {
    // ---------------- epilogue: TMEM lane quadrant = warp % 4, column half = (warp - 2) / 4; a thread owns one row ----------------
    const int quad = warp & 3, half = (warp - 2) >> 2;
    int buf = 0;
    uint32_t tphase = 0;
    bool ok = true;
    float g = 1.f;
    if (EPI == EPI_OUT) g = p.scale * (p.grad_out ? *p.grad_out : 1.f) * (p.inv_live ? *p.inv_live : 1.f);
    // rows of the output on 32-byte boundaries: each thread stores its own; else they pass through shared memory
    const bool vec = p.width % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;
    constexpr int BOXES = C::OUT_BYTES / (EPI_WARPS * OUT_BOX_BYTES);
    unsigned char* boxes = sOut + (warp - 2) * BOXES * OUT_BOX_BYTES;
    int box_at = 0;
    // 16-byte unit `unit` (of 8) of row r of the box in turn, where the tensor map's swizzle has it
    auto box_unit = [&](int r, int unit) { return boxes + box_at + r * 128 + ((unit ^ (r & 7)) << 4); };
    auto box_put = [&](int c0, const uint32_t(&o)[16]) {   // the lane's row, 32 elements from column c0 (0 or 32)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4*>(box_unit(lane, (c0 >> 3) + q)) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
    };
    auto box_open = [&]() {   // the box before the last has left
      if (lane == 0) tma_store_wait_read<1>();
      __syncwarp();
    };
    auto box_send = [&](int x, int y) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) tma_store_2d(&tmOut, smem_u32(boxes + box_at), x, y);
      box_at ^= OUT_BOX_BYTES;
    };
    const uint32_t acc_mask = d.kb > 0 ? 0xffffffffu : 0u;   // no live rows: the accumulator holds stale values
    while (ok && walk.step()) {
      const Tile tl = decode<FORM, CTA2>(p, d, walk.t, rank);
      const int row = tl.mt * BM + quad * 32 + lane;
      const bool row_live = row < d.m;
      const int col_first = tl.nt * BN + half * (BN / 2);
      const int left = d.n - col_first;   // columns of this half tile that exist
      // dW sums over blocks of BK rows: of dz, the rows up to that boundary are wanted, as zeros behind the last live one
      const int rows_wanted = EPI == EPI_PROB ? (d.m + BK - 1) / BK * BK : d.m;
      const bool idle = tl.mt * BM + quad * 32 >= rows_wanted || left <= 0 && EPI == EPI_OUT;   // nothing for this warp
      float off = 0.f, diff = 0.f;
      long long out_row = row;
      int want = -1;                      // column of the row's target in this half tile
      if (EPI == EPI_PROB && row_live) {
        off = p.shift - p.lse2[row];
        if (p.tgt) {
          want = p.tgt[row] - p.class0 - col_first;
          diff = p.tdiff[row];
        }
      }
      if (EPI == EPI_OUT && row_live) out_row = p.row_map ? p.row_map[row] : (long long)p.class0 + row;
      if (EPI == EPI_LSE && row_live) want = p.tgt[row] - col_first;
      ok = mbar_wait(bar_tfull + 8 * buf, (tphase >> buf) & 1, abort_flag, p.status, 14);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + half * (BN / 2));
      auto release = [&]() {   // the accumulator may be overwritten once every epilogue warp (of both CTAs) has read it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CTA2) mbar_arrive_cluster_tmem(cluster_addr(bar_tempty + 8 * buf, 0)); else mbar_arrive(bar_tempty + 8 * buf);
        }
        tphase ^= 1u << buf;
        buf ^= 1;
      };
      // f(first column, 32 values) for the half tile's four chunks; the next chunk is on its way while one is worked on, and the accumulator
      // goes back before the last one is
      auto chunks = [&](auto&& f) {
        uint32_t a[32], b[32];
        tmem_ld32_async(taddr, a);
        tmem_wait(a);
        tmem_ld32_async(taddr + 32, b);
        f(0, a);
        __syncwarp();
        tmem_wait(b);
        tmem_ld32_async(taddr + 64, a);
        f(32, b);
        __syncwarp();
        tmem_wait(a);
        tmem_ld32_async(taddr + 96, b);
        f(64, a);
        __syncwarp();
        tmem_wait(b);
        release();
        f(96, b);
      };
      if (idle) {
        release();
        continue;
      }
      if (EPI == EPI_LSE) {
        // the few targets in this half tile
        unsigned hits = __ballot_sync(0xffffffffu, want >= 0 && want < BN / 2);
        while (hits) {
          const int owner = __ffs(hits) - 1, col = __shfl_sync(0xffffffffu, want, owner);
          const uint32_t z = tmem_ld1(taddr + col);
          if (lane == owner) p.zt[row] = __uint_as_float(z);
          __syncwarp();
          hits &= hits - 1;
        }
        float m = -1e30f, s = 0.f;   // maximum of z and sum of 2^((z - m) c)
        chunks([&](int c0, uint32_t(&r)[32]) {
          if (left < c0 + 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = c0 + i < left ? r[i] : 0xff800000u;
          }
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(r[i]), __uint_as_float(r[i + 4]));
#pragma unroll
          for (int i = 8; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(r[i]));
          const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), m);
          s *= ex2f((m - top) * p.c);
          m = top;
          const f32x2 cc = splat2(p.c), mc = splat2(-m * p.c);
          f32x2 sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x, y;
            unpack2(fma2(pack2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), cc, mc), x, y);
            sum[(i >> 1) & 3] = add2(sum[(i >> 1) & 3], pack2(ex2f(x), ex2f(y)));
          }
          float x, y;
          unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), x, y);
          s += x + y;
        });
        if (row_live) p.part[(long long)(2 * tl.nt + half) * p.part_ld + row] = make_float2(m * p.c, s);
      } else if (EPI == EPI_PROB) {
        const uint32_t keep = row_live ? 0xffffffffu : 0u;
        chunks([&](int c0, uint32_t(&r)[32]) {
          uint32_t o[16];
          const f32x2 cc = splat2(p.c), oo = splat2(off);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x, y;
            unpack2(fma2(pack2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), cc, oo), x, y);
            o[i >> 1] = pack_pair<T>(ex2f(x), ex2f(y)) & keep;
          }
          if (left < c0 + 32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int have = left - c0 - 2 * i;
              o[i] &= have >= 2 ? 0xffffffffu : (have == 1 ? 0x0000ffffu : 0u);
            }
          }
          if (!(c0 & 32)) box_open();
          box_put(c0 & 32, o);
          if (c0 & 32) {
            const int at = want - (c0 & 64);
            if (at >= 0 && at < 64) *reinterpret_cast<T*>(box_unit(lane, at >> 3) + (at & 7) * 2) = Num<T>::from_f(diff);   // rounded once
            box_send(col_first + (c0 & 64), tl.mt * BM + quad * 32);
          }
        });
      } else if (walk.slot >= 0 || (ACC && p.acc_out)) {
        // float32 results: a part of a split tile, or the sums over the pieces so far (row strides of whole tiles: no bounds)
        const bool part = walk.slot >= 0;
        float* dst = part ? p.slots + ((long long)walk.slot * (CTA2 ? 2 * BM : BM) + rank * BM + quad * 32 + lane) * BN + half * (BN / 2)
                          : p.acc + row * p.acc_ld + col_first;
        const bool add = ACC && !part && p.acc_in;
        chunks([&](int c0, uint32_t(&r)[32]) {
          if (!row_live) return;
          if (add) {
#pragma unroll
            for (int q = 0; q < 32; q += 4) {
              const float4 x = *reinterpret_cast<const float4*>(dst + c0 + q);
              r[q] = __float_as_uint(__uint_as_float(r[q]) + x.x);
              r[q + 1] = __float_as_uint(__uint_as_float(r[q + 1]) + x.y);
              r[q + 2] = __float_as_uint(__uint_as_float(r[q + 2]) + x.z);
              r[q + 3] = __float_as_uint(__uint_as_float(r[q + 3]) + x.w);
            }
          }
#pragma unroll
          for (int q = 0; q < 32; q += 8)
            st_global_32B(dst + c0 + q, make_uint4(r[q], r[q + 1], r[q + 2], r[q + 3]),
                          make_uint4(r[q + 4], r[q + 5], r[q + 6], r[q + 7]));
        });
      } else {
        T* dst = static_cast<T*>(p.out) + out_row * p.width + col_first;
        chunks([&](int c0, uint32_t(&r)[32]) {
          if (left <= (c0 & 64)) return;   // the same for the whole warp
          uint32_t o[16];
          if (ACC) {
            const float* acc = p.acc + row * p.acc_ld + col_first + c0;
            if (row_live) {
#pragma unroll
              for (int q = 0; q < 32; q += 4) {
                const float4 x = *reinterpret_cast<const float4*>(acc + q);
                r[q] = __float_as_uint(__uint_as_float(r[q]) + x.x);
                r[q + 1] = __float_as_uint(__uint_as_float(r[q + 1]) + x.y);
                r[q + 2] = __float_as_uint(__uint_as_float(r[q + 2]) + x.z);
                r[q + 3] = __float_as_uint(__uint_as_float(r[q + 3]) + x.w);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            o[i >> 1] = pack_pair<T>(__uint_as_float(r[i] & acc_mask) * g, __uint_as_float(r[i + 1] & acc_mask) * g);
          if (p.boxes) {
            if (!(c0 & 32)) box_open();
            box_put(c0 & 32, o);
            if (c0 & 32) box_send(col_first + (c0 & 64), p.class0 + tl.mt * BM + quad * 32);
            return;
          }
          if (vec && left >= (c0 & 64) + 64) {
            if (row_live) {
#pragma unroll
              for (int q = 0; q < 16; q += 8)
                st_global_32B(dst + c0 + 2 * q, make_uint4(o[q], o[q + 1], o[q + 2], o[q + 3]),
                              make_uint4(o[q + 4], o[q + 5], o[q + 6], o[q + 7]));
            }
            return;
          }
          // rows on other boundaries: the warp's 32 x 64 block through a box, then row by row in neighbouring lanes, 4 bytes each; a row
          // that starts between 4-byte boundaries goes out as its first element, words across the staged ones, and its last element
          box_put(c0 & 32, o);
          if (!(c0 & 32)) return;
          __syncwarp();
          const int cols = min(64, left - (c0 & 64)), rows = min(32, d.m - (tl.mt * BM + quad * 32));
          const unsigned long long mine = reinterpret_cast<unsigned long long>(dst + (c0 & 64));
          const unsigned long long first = __shfl_sync(0xffffffffu, mine, 0);
#pragma unroll 1
          for (int r0 = 0; r0 < rows; r0 += 8) {   // eight rows' words first, then their stores
            uint32_t word[8], next[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) word[j] = *reinterpret_cast<const uint32_t*>(box_unit(r0 + j, lane >> 2) + (lane & 3) * 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) next[j] = __shfl_down_sync(0xffffffffu, word[j], 1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int r = r0 + j;
              unsigned char* to = reinterpret_cast<unsigned char*>(p.row_map ? __shfl_sync(0xffffffffu, mine, r)
                                                                             : first + (unsigned long long)(2 * r) * p.width);
              const int odd = (reinterpret_cast<uintptr_t>(to) >> 1) & 1;      // elements before the first 4-byte boundary
              const uint32_t out = odd ? __funnelshift_r(word[j], next[j], 16) : word[j];
              const int e = r < rows ? 2 * lane + odd : OUT_COLS;              // first of this lane's two elements
              if (e == 1 && lane == 0) *reinterpret_cast<uint16_t*>(to) = (uint16_t)word[j];
              if (e + 1 < cols) *reinterpret_cast<uint32_t*>(to + 2 * e) = out;
              if (e + 1 == cols) *reinterpret_cast<uint16_t*>(to + 2 * e) = (uint16_t)out;
            }
          }
          __syncwarp();
        });
      }
    }
    if (lane == 0) tma_store_wait();   // the last boxes are in place before the kernel ends
  }
  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up: let TMA copies that may still be in flight land before the CTA goes away
    const unsigned long long t0 = now_ns();
    while (now_ns() - t0 < 200000ull) {
    }
    __syncthreads();
  }
  if (CTA2) cluster_sync_all();   // the peer no longer signals this CTA's barriers or reads its shared memory
  if (warp == 1) {
    tc_fence_after();
    if (CTA2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// Adds the parts of split tiles in a fixed order and finishes them as the product's epilogue does; a thread takes four columns.  Where tiles have
// many parts (few rows) a block takes one row and its four groups of threads share the parts, else each group has rows of its own (captured
// passes, one row / 16 rows a block: 64 x 50257 x 512 78 / 137 us, 1000 x 6112 x 2080 161 / 140).
constexpr int JOIN_ROWS = 16, JOIN_MANY = 8;
struct JoinTile {
  int mu, nt, w0, w1, late;   // unit, column tile; first and last worker with a part; whether the first one's is its second part
};
template <typename T, int FORM, bool CTA2>
__global__ void __launch_bounds__(256) join_tiles_kernel(Params p, int workers, int rows_per_block) {
  chain_enter();
  __shared__ float4 s_part[4][64];
  __shared__ JoinTile s_tile;
  const Dims d = dims_of<FORM, CTA2>(p);
  if (threadIdx.x == 0) {
    const Split s = split_of(d.mu * d.nt, d.kb, workers);
    JoinTile jt = {0, 0, 0, -1, 0};   // no parts
    const int j = blockIdx.x;
    if (j < s.rem) {
      decode_unit<FORM, CTA2>(p, d, s.full + j, jt.mu, jt.nt);
      const long long a = (long long)j * s.kb, b = a + s.kb;
      jt.w0 = (int)(a * s.parts / s.iters);
      while (jt.w0 > 0 && s.begin(jt.w0) > a) --jt.w0;
      while (s.begin(jt.w0 + 1) <= a) ++jt.w0;
      jt.w1 = (int)((b - 1) * s.parts / s.iters);
      while (jt.w1 > 0 && s.begin(jt.w1) > b - 1) --jt.w1;
      while (s.begin(jt.w1 + 1) <= b - 1) ++jt.w1;
      jt.late = s.begin(jt.w0) < a;
      if (jt.w0 == jt.w1 && !jt.late && s.begin(jt.w0 + 1) == b) jt.w1 = -1;   // one worker had all of it
    }
    s_tile = jt;
  }
  __syncthreads();
  const JoinTile jt = s_tile;
  constexpr int UNIT = CTA2 ? 2 * BM : BM;
  const int row0 = blockIdx.y * rows_per_block;
  if (jt.w1 < 0 || jt.mu * UNIT + row0 >= d.m) return;
  const float g = p.scale * (p.grad_out ? *p.grad_out : 1.f) * (p.inv_live ? *p.inv_live : 1.f);
  const int col = (threadIdx.x & 63) * 4, grp = threadIdx.x >> 6;
  const int n0 = jt.nt * BN + col;
  auto sum = [&](int i, int from, int step) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int w = from; w <= jt.w1; w += step) {
      const int slot = 2 * w + (w == jt.w0 ? jt.late : 0);
      const float4 x = *reinterpret_cast<const float4*>(p.slots + ((long long)slot * UNIT + i) * BN + col);
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    return v;
  };
  auto finish = [&](int i, const float4& x) {
    const int row = jt.mu * UNIT + i;
    const float v[4] = {x.x, x.y, x.z, x.w};
    float* acc = p.acc + row * p.acc_ld + n0;
    T* out = static_cast<T*>(p.out) + (p.row_map ? p.row_map[row] : (long long)p.class0 + row) * p.width + n0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (n0 + c >= d.n) break;
      const float t = p.acc && p.acc_in ? v[c] + acc[c] : v[c];
      if (p.acc && p.acc_out)
        acc[c] = t;
      else
        out[c] = Num<T>::from_f(t * g);
    }
  };
  if (rows_per_block == JOIN_ROWS) {
    constexpr int N = JOIN_ROWS / 4;
    float4 v[N];
#pragma unroll
    for (int o = 0; o < N; ++o)
      if (jt.mu * UNIT + row0 + 4 * o + grp < d.m) v[o] = sum(row0 + 4 * o + grp, jt.w0, 1);
#pragma unroll
    for (int o = 0; o < N; ++o)
      if (jt.mu * UNIT + row0 + 4 * o + grp < d.m) finish(row0 + 4 * o + grp, v[o]);
    return;
  }
  s_part[grp][threadIdx.x & 63] = sum(row0, jt.w0 + grp, 4);
  __syncthreads();
  if (grp == 0) {
    float4 v = s_part[0][threadIdx.x];
    for (int q = 1; q < 4; ++q) {
      const float4 x = s_part[q][threadIdx.x];
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    finish(row0, v);
  }
}

// ---- live rows ------------------------------------------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// One row of 16-bit elements by one warp to a destination on a 16-byte boundary: 16 bytes a lane where the source allows it, else 4-byte words,
// put together from two where the source lies between 4-byte boundaries.
__device__ __forceinline__ void copy_row(uint16_t* __restrict__ dst, const uint16_t* __restrict__ src, int width) {
  const int lane = threadIdx.x & 31;
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int nv = width / 8;
#pragma unroll 4
    for (int i = lane; i < nv; i += 32) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
    done = nv * 8;
  } else {
    const int off = (reinterpret_cast<uintptr_t>(src) >> 1) & 1;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(src - off);
    const int nw = (width - off) / 2;   // the last word read ends inside the row
    constexpr int N = 8;
    for (int i0 = lane; i0 < nw; i0 += 32 * N) {   // all loads of a round before its stores
      uint32_t a[N], b[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        a[n] = i0 + 32 * n < nw ? words[i0 + 32 * n] : 0u;
        b[n] = off && i0 + 32 * n < nw ? words[i0 + 32 * n + 1] : 0u;
      }
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (i0 + 32 * n < nw) reinterpret_cast<uint32_t*>(dst)[i0 + 32 * n] = off ? __funnelshift_r(a[n], b[n], 16) : a[n];
    }
    done = nw * 2;
  }
  for (int i = done + lane; i < width; i += 32) dst[i] = src[i];
}
// Zeros for a row on any boundary.
__device__ __forceinline__ void zero_row(uint16_t* dst, int width) {
  const int lane = threadIdx.x & 31;
  const int head = min(width, (int)(((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / 2));
  const int nv = (width - head) / 8;
  if (lane < head) dst[lane] = 0;
  for (int i = lane; i < nv; i += 32) reinterpret_cast<uint4*>(dst + head)[i] = make_uint4(0, 0, 0, 0);
  for (int i = head + nv * 8 + lane; i < width; i += 32) dst[i] = 0;
}

__device__ __forceinline__ bool row_is_live(const long long* target, const int32_t* flags, int r, int vocab) {
  if (flags) return flags[r] != 0;
  const long long t = target[r];
  return t >= 0 && t < vocab;
}

// Packs the live rows: pos[r] = packed index of row r or -1, pos[rows] = their number, packed rows.  Each block owns a range of rows and first
// counts the live rows before it.  What the buffer holds behind them reaches only results that no one keeps.
__global__ void __launch_bounds__(kRowThreads)
pack_rows_kernel(const uint16_t* __restrict__ hidden, long long ld, const long long* __restrict__ target, const int32_t* __restrict__ flags,
                 const int32_t* __restrict__ top, int rows, int vocab, int width, uint16_t* __restrict__ packed, int packed_ld, int32_t* __restrict__ origin,
                 int32_t* __restrict__ tgt, int32_t* __restrict__ pos, float* __restrict__ loss_rows, float* __restrict__ lse_rows,
                 int* __restrict__ done) {
  chain_enter();
  if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;   // blocks of the forward pass's last kernel that have ended
  __shared__ int s_warp[kRowThreads / 32];
  __shared__ int s_at[kRowThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (rows + gridDim.x - 1) / gridDim.x;
  const int r0 = min(rows, (int)blockIdx.x * per), r1 = min(rows, r0 + per);
  int before = 0;
  for (int r = threadIdx.x; r < r0; r += kRowThreads) before += row_is_live(target, flags, r, vocab);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
  if (lane == 0) s_warp[warp] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < kRowThreads / 32; ++w) before += s_warp[w];
  for (int base = r0; base < r1; base += kRowThreads) {
    __syncthreads();
    const int r = base + threadIdx.x;
    const bool live = r < r1 && row_is_live(target, flags, r, vocab);
    const unsigned ballot = __ballot_sync(0xffffffffu, live);
    if (lane == 0) s_warp[warp] = __popc(ballot);
    __syncthreads();
    int at = before;
    for (int w = 0; w < warp; ++w) at += s_warp[w];
    at += __popc(ballot & ((1u << lane) - 1));
    if (r < r1) {
      pos[r] = live ? at : -1;
      if (live) {
        origin[at] = r;
        tgt[at] = target ? (int)target[r] : top[r];
      } else {
        loss_rows[r] = 0.f;
        lse_rows[r] = 0.f;
      }
    }
    s_at[threadIdx.x] = live ? at : -1;
    __syncthreads();
    for (int i = warp; i < min(kRowThreads, r1 - base); i += kRowThreads / 32)
      if (s_at[i] >= 0) copy_row(packed + (long long)s_at[i] * packed_ld, hidden + (long long)(base + i) * ld, width);
    for (int w = 0; w < kRowThreads / 32; ++w) before += s_warp[w];
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) pos[rows] = before;
}

// Rows to a padded row stride (a weight whose rows a tensor map cannot describe).
__global__ void __launch_bounds__(kRowThreads)
copy_rows_kernel(const uint16_t* __restrict__ src, long long lds, uint16_t* __restrict__ dst, long long ldd, int rows, int width) {
  chain_enter();
  const int warps = gridDim.x * (kRowThreads / 32);
  for (int r = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5); r < rows; r += warps) copy_row(dst + r * ldd, src + r * lds, width);
}

// The same packing in the backward pass, from pos; gradient rows of ignored rows are zeroed, lse goes to packed order and base 2.  dW sums over
// blocks of BK rows: the last one is filled up with zeros (dz has zeros there, but 0 x NaN would remain).
__global__ void __launch_bounds__(kRowThreads)
repack_rows_kernel(const uint16_t* __restrict__ hidden, long long ld, const int32_t* __restrict__ pos, const float* __restrict__ lse_rows,
                   const long long* __restrict__ target, const float* __restrict__ loss_rows, float unit, int rows, int width,
                   uint16_t* __restrict__ packed, int packed_ld, int32_t* __restrict__ origin, float* __restrict__ lse2,
                   int32_t* __restrict__ tgt, float* __restrict__ tdiff, uint16_t* __restrict__ dhidden) {
  chain_enter();
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (kRowThreads / 32);
  const int first = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  for (int r = first; r < rows; r += warps) {
    const int at = pos[r];
    if (at >= 0) {
      copy_row(packed + (long long)at * packed_ld, hidden + (long long)r * ld, width);
      if (lane == 0) {
        origin[at] = r;
        lse2[at] = lse_rows[r] * kLog2e;
        if (target) {
          tgt[at] = (int)target[r];
          tdiff[at] = expm1f(-loss_rows[r]) * unit;   // probability of the target less 1
        }
      }
    } else if (dhidden) {
      zero_row(dhidden + (long long)r * width, width);
    }
  }
  const int count = pos[rows], end = (count + BK - 1) / BK * BK;
  for (int i = count + first; i < end; i += warps) zero_row(packed + (long long)i * packed_ld, width);
}

// ---- row results ----------------------------------------------------------------------------------------------------------
constexpr int kFinishThreads = 256;

// Dot product of two rows by LANES neighbouring lanes; all of them get it.  Both rows start on 16-byte boundaries (packed rows; the weight's rows
// as the tensor map wants them).
template <typename T, int LANES, int N>
__device__ __forceinline__ void group_dots(const T* __restrict__ a, const T* const* b, int width, float* out) {
  const int sub = threadIdx.x & (LANES - 1);
  float s[N];
#pragma unroll
  for (int n = 0; n < N; ++n) s[n] = 0.f;
  const int nv = width / 8;
#pragma unroll 4
  for (int i = sub; i < nv; i += LANES) {
    const uint4 x = reinterpret_cast<const uint4*>(a)[i];
    uint4 y[N];
#pragma unroll
    for (int n = 0; n < N; ++n) y[n] = reinterpret_cast<const uint4*>(b[n])[i];
    const T* xs = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const T* ys = reinterpret_cast<const T*>(&y[n]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[n] = fmaf(Num<T>::to_f(xs[j]), Num<T>::to_f(ys[j]), s[n]);
    }
  }
  for (int i = nv * 8 + sub; i < width; i += LANES)
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = fmaf(Num<T>::to_f(a[i]), Num<T>::to_f(b[n][i]), s[n]);
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] += __shfl_xor_sync(0xffffffffu, s[n], d);
#pragma unroll
  for (int n = 0; n < N; ++n) out[n] = s[n];
}

struct FinishArgs {
  const float2* part;      // [n_part][part_ld] maxima and sums of the column half tiles
  long long part_ld;
  int n_part;
  const int32_t* count;
  const int32_t* origin;
  const void* packed;
  int packed_ld;
  const void* weight;
  long long weight_ld;
  int width;
  const int32_t* tgt;      // targets (or the teachers' likeliest classes) and their logits from the product, by packed row
  const float* zt;
  const int32_t* idx;      // teachers: classes (-1: none), q, class weights, [rows][k]
  const float* q;
  const float* cw;
  int k;
  float inv_t;
  float *loss_rows, *lse_rows, *diff;
  double* block_sums;
  int* done;
  float *mean, *inv_live;
};

// A block finishes kRows packed rows: joins the partial maxima and sums of its rows' column half tiles (in a fixed order), and computes the
// logits at the rows' targets, or at the entries of their teachers, as float32 dot products.  The tensor cores cut the sums of products short (at
// a logit of 12 of 1024 products 1e-5 low where they have both signs, 8e-5 where all are positive), which the loss would show where a target (or
// a teacher's likeliest class) holds most of the probability: its share of the row's sum is replaced by the dot product's.  The other classes
// keep what was cut: a common offset of 100 in all logits makes the loss 1.4e-4 low at width 1024 (6e-4 at 4096), about what float32 logits
// scatter by (1.3e-4, 2.8e-4).  The dot product of the target takes a warp and is under way before the sums are joined; a teacher's entries take
// eight lanes each, two at a time.
template <typename T, int kRows, bool TEACHER>
__global__ void __launch_bounds__(kFinishThreads, TEACHER ? 3 : 5)
finish_rows_kernel(FinishArgs a) {
  chain_enter();
  constexpr int G = kFinishThreads / kRows, W = kFinishThreads / 32;
  static_assert(kRows <= W, "a warp per row");
  extern __shared__ float s_terms[];   // TEACHER: [kRows][k] terms of the sums
  __shared__ float s_m[W][kRows], s_s[W][kRows];
  __shared__ float s_lse[kRows], s_loss[kRows];
  const int n = *a.count;
  const int base = blockIdx.x * kRows;
  const int live = max(0, min(kRows, n - base));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rr = threadIdx.x % kRows, grp = threadIdx.x / kRows;
  const T* packed = static_cast<const T*>(a.packed);
  const T* weight = static_cast<const T*>(a.weight);
  float z = 0.f, z_product = 0.f;
  if (warp < live) {
    const int c = base + warp;
    const T* b[1] = {weight + (long long)a.tgt[c] * a.weight_ld};
    group_dots<T, 32, 1>(packed + (long long)c * a.packed_ld, b, a.width, &z);
    z_product = a.zt[c];
  }
  float m = -1e38f, s = 0.f;
  auto merge = [&](float m2, float s2) {
    const float mm = fmaxf(m, m2);
    s = s * ex2f(m - mm) + s2 * ex2f(m2 - mm);
    m = mm;
  };
  if (rr < live) {
#pragma unroll 4
    for (int t = grp; t < a.n_part; t += G) {
      const float2 v = a.part[(long long)t * a.part_ld + base + rr];
      merge(v.x, v.y);
    }
  }
#pragma unroll
  for (int d = kRows; d < 32; d <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, d), s2 = __shfl_xor_sync(0xffffffffu, s, d);
    merge(m2, s2);
  }
  if (lane < kRows) {
    s_m[warp][lane] = m;
    s_s[warp][lane] = s;
  }
  __syncthreads();
  if ((int)threadIdx.x < live) {
    m = s_m[0][threadIdx.x];
    s = s_s[0][threadIdx.x];
    for (int w = 1; w < W; ++w) merge(s_m[w][threadIdx.x], s_s[w][threadIdx.x]);
    s_lse[threadIdx.x] = m * kLn2 + logf(s);
  }
  __syncthreads();
  if (warp < live && lane == 0) {   // warp w has the dot product of row w
    const float lse = s_lse[warp];
    s_lse[warp] = lse + log1pf(expf(z_product * a.inv_t - lse) * expm1f((z - z_product) * a.inv_t));
  }
  if (!TEACHER) {
    if (warp < live && lane == 0) {
      const int r = a.origin[base + warp];
      a.loss_rows[r] = s_loss[warp] = s_lse[warp] - z;
      a.lse_rows[r] = s_lse[warp];
    }
  } else {
    __syncthreads();
    const int pairs = (a.k + 1) / 2, sub = lane & 7;
    for (int t0 = warp * 4; t0 < live * pairs; t0 += W * 4) {   // four pairs of entries per warp
      const int t = min(t0 + (lane >> 3), live * pairs - 1);
      const int i = t / pairs, e0 = (t - i * pairs) * 2, c = base + i;
      const long long at = (long long)a.origin[c] * a.k;
      const bool two = e0 + 1 < a.k;
      const int cls[2] = {a.idx[at + e0], two ? a.idx[at + e0 + 1] : -1};
      const T* b[2] = {weight + (long long)max(cls[0], 0) * a.weight_ld, weight + (long long)max(cls[1], 0) * a.weight_ld};
      float zs[2];
      group_dots<T, 8, 2>(packed + (long long)c * a.packed_ld, b, a.width, zs);
      if (sub < 2 && (sub == 0 || two)) {
        const int e = e0 + sub;
        const bool counts = cls[sub] >= 0;
        const float lp = (sub ? zs[1] : zs[0]) * a.inv_t - s_lse[i], qe = a.q[at + e];
        s_terms[i * a.k + e] = counts && qe != 0.f ? qe * (logf(qe) - lp) : 0.f;
        a.diff[at + e] = counts ? expf(lp) - a.cw[at + e] : 0.f;
      }
    }
    __syncthreads();
    for (int i = warp; i < live; i += W) {
      float sum = 0.f;
      for (int e = lane; e < a.k; e += 32) sum += s_terms[i * a.k + e];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) {
        const int r = a.origin[base + i];
        a.loss_rows[r] = s_loss[i] = sum / (a.inv_t * a.inv_t);
        a.lse_rows[r] = s_lse[i];
      }
    }
  }
  // the block that ends last takes the mean: the blocks' sums in one order, in 64 bits
  __shared__ bool s_last;
  __shared__ double s_sum[W];
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < live; ++i) sum += (double)s_loss[i];
    a.block_sums[blockIdx.x] = sum;
    __threadfence();
    s_last = atomicAdd(a.done, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
#pragma unroll 4
  for (int b = threadIdx.x; b < (int)gridDim.x; b += kFinishThreads) sum += __ldcg(a.block_sums + b);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < W; ++w) sum += s_sum[w];
    const int div = n > 1 ? n : 1;
    *a.mean = (float)(sum / div);
    *a.inv_live = 1.0f / (float)div;
  }
}

// Teacher distributions of all rows, a warp each: q, class weights, indices as int32 (-1: does not count), the class of the largest q, live
// flags.
constexpr int kTeacherWarps = 4;
__global__ void __launch_bounds__(32 * kTeacherWarps)
teacher_kernel(const void* __restrict__ values, int vdtype, const long long* __restrict__ indices, int rows, int k, float inv_t, int vocab,
               float* __restrict__ q, float* __restrict__ cw, int32_t* __restrict__ idx, int32_t* __restrict__ top, int32_t* __restrict__ live) {
  chain_enter();
  __shared__ float s_q[kTeacherWarps][kMaxTop];
  __shared__ int s_idx[kTeacherWarps][kMaxTop];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r = (long long)blockIdx.x * kTeacherWarps + warp;
  if (r >= rows) return;
  const bool alive = teacher_row(values, vdtype, indices, r, k, inv_t, vocab, s_q[warp], s_idx[warp]);
  float best = -1.f;   // largest q and its class; rows with NaN keep class 0
  int cls = 0;
  for (int i = lane; i < k; i += 32)
    if (s_idx[warp][i] >= 0 && s_q[warp][i] > best) {
      best = s_q[warp][i];
      cls = s_idx[warp][i];
    }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float b2 = __shfl_xor_sync(0xffffffffu, best, d);
    const int c2 = __shfl_xor_sync(0xffffffffu, cls, d);
    if (b2 > best || (b2 == best && c2 < cls)) {
      best = b2;
      cls = c2;
    }
  }
  if (lane == 0) {
    live[r] = alive;
    top[r] = cls;
  }
  for (int i = lane; i < k; i += 32) {
    q[r * k + i] = s_q[warp][i];
    cw[r * k + i] = class_weight(s_q[warp], s_idx[warp], k, i);
    idx[r * k + i] = s_idx[warp][i];
  }
}

// dz at the teacher's classes of the piece: the difference in float32, rounded once.  Entries of one row that name the same class write the
// same value.
template <typename T>
__global__ void __launch_bounds__(256)
place_targets_kernel(const int32_t* __restrict__ count, const int32_t* __restrict__ origin, const long long* __restrict__ top_indices,
                     const float* __restrict__ diff, int k, int class0, int classes, float unit, T* __restrict__ dz, long long dz_ld) {
  chain_enter();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long c = i / k;
  if (c >= *count) return;
  const long long e = (long long)origin[c] * k + (i - c * k);
  const long long at = top_indices[e] - class0;
  if (at >= 0 && at < classes) dz[c * dz_ld + at] = Num<T>::from_f(diff[e] * unit);
}

// ---- host side ------------------------------------------------------------------------------------------------------------
static int make_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, int dtype) {
  EncodeTiledFn fn = encode_fn();
  LANCET_REQUIRE(fn, LANCET_ERR_CUDA, "head product: the driver does not provide cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)BK, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, dtype == LANCET_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                  const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LANCET_REQUIRE(r == CUDA_SUCCESS, LANCET_ERR_CUDA, "head product: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return LANCET_OK;
}

// The paired form halves the bytes of B through shared memory per product; up to 128 rows its second tile would be empty (captured passes at
// 50257 x 1024, one CTA / pairs: 100 rows 129 / 130 us, 200 rows 171 / 143, 511 rows 267 / 218; 4096 x 32000 x 2048 1.67 / 1.47 ms).
static bool paired_for(int m) { return m > BM; }

template <typename T, int FORM, int EPI, bool CTA2, bool ACC>
static int launch_form(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmOut, const Params& p, long long units, bool split,
                       int* workers, cudaStream_t st) {
  auto kernel = head_product_kernel<T, FORM, EPI, CTA2, ACC>;
  constexpr int SMEM = Cfg<FORM, EPI, CTA2>::SMEM_BYTES;
  static int set_for[64] = {0};   // per device
  int dev = 0;
  LANCET_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !__atomic_load_n(&set_for[dev], __ATOMIC_ACQUIRE)) {
    LANCET_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev >= 0 && dev < 64) __atomic_store_n(&set_for[dev], 1, __ATOMIC_RELEASE);
  }
  long long grid = sm_count();
  if (gemm_cta_limit() > 0 && gemm_cta_limit() < grid) grid = gemm_cta_limit();
  if (!split && grid > units * (CTA2 ? 2 : 1)) grid = units * (CTA2 ? 2 : 1);
  if (CTA2) grid &= ~1ll;
  if (grid < (CTA2 ? 2 : 1)) grid = CTA2 ? 2 : 1;
  *workers = (int)grid / (CTA2 ? 2 : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = chained_launch_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTA2 ? 2 : 1;
  {
    ProfScope prof("head_product_kernel", st);
    cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, tmOut, p);
  }
  return launch_status("head_product_kernel");
}

template <typename T, int FORM, int EPI, bool CTA2>
static int launch_product_as(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmOut, const Params& p, int m, int n, int k,
                             cudaStream_t st) {
  constexpr int UNIT = CTA2 ? 2 * BM : BM;
  const long long units = ((long long)(m + UNIT - 1) / UNIT) * ((n + BN - 1) / BN);
  LANCET_REQUIRE(units < (1ll << 30), LANCET_ERR_INVALID, "head product: %lld tiles", units);
  const bool split = EPI == EPI_OUT && (k + BK - 1) / BK > SPLIT_MIN_KB;   // the least length of a reduction that split_of cuts
  int workers = 0;
  if constexpr (FORM == FORM_DH) {
    if (p.acc) {
      if (int rc = launch_form<T, FORM, EPI, CTA2, true>(tmA, tmB, tmOut, p, units, split, &workers, st)) return rc;
    } else if (int rc = launch_form<T, FORM, EPI, CTA2, false>(tmA, tmB, tmOut, p, units, split, &workers, st)) {
      return rc;
    }
  } else if (int rc = launch_form<T, FORM, EPI, CTA2, false>(tmA, tmB, tmOut, p, units, split, &workers, st)) {
    return rc;
  }
  if constexpr (EPI == EPI_OUT) {
    if (split) {
      const int most = (int)(units < workers ? units : workers);   // tiles that can have been cut
      const int per = workers >= JOIN_MANY * units ? 1 : JOIN_ROWS;
      const int rows = m < UNIT ? m : UNIT;
      launch_chained(join_tiles_kernel<T, FORM, CTA2>, dim3(most, (rows + per - 1) / per), dim3(256), 0, st, p, workers, per);
      return launch_status("join_tiles_kernel");
    }
  }
  return LANCET_OK;
}
// m, n, k: upper bounds of the product's sizes (the live rows are known on the device only)
template <typename T, int FORM, int EPI>
static int launch_product(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmOut, const Params& p, int m, int n, int k,
                          bool paired, cudaStream_t st) {
  return paired ? launch_product_as<T, FORM, EPI, true>(tmA, tmB, tmOut, p, m, n, k, st)
                : launch_product_as<T, FORM, EPI, false>(tmA, tmB, tmOut, p, m, n, k, st);
}

struct Carver {
  char* base;
  size_t used = 0;
  explicit Carver(void* p) : base(static_cast<char*>(p)) {}
  template <typename U>
  U* take(size_t n) {
    used = (used + 255) / 256 * 256;
    U* p = base ? reinterpret_cast<U*>(base + used) : nullptr;
    used += n * sizeof(U);
    return p;
  }
};

static long long pad_rows(long long rows) { return rows < 1 ? ROW_PAD : (rows + ROW_PAD - 1) / ROW_PAD * ROW_PAD; }
static long long pad_cols(int width) { return (width + BN - 1) / BN * BN; }
static int pad_width(int width) { return (width + 7) / 8 * 8; }

struct FwdWs {
  uint16_t* packed;
  int32_t* origin;
  float2* part;
  int32_t* tgt;
  int* done;
  double* block_sums;
  float* zt;
  float* q;
  float* cw;
  int32_t* idx;
  int32_t* top;
  int32_t* live;
  size_t bytes;
};
static FwdWs fwd_ws(void* ws, int rows, int vocab, int width, int k) {
  Carver c(ws);
  FwdWs w;
  w.packed = c.take<uint16_t>((size_t)pad_rows(rows) * pad_width(width));
  w.origin = c.take<int32_t>(rows);
  w.part = c.take<float2>((size_t)2 * ((vocab + BN - 1) / BN) * pad_rows(rows));
  w.tgt = c.take<int32_t>(rows);
  w.zt = c.take<float>(rows);
  w.done = c.take<int>(1);
  w.block_sums = c.take<double>(rows);
  w.q = c.take<float>((size_t)rows * k);
  w.cw = c.take<float>((size_t)rows * k);
  w.idx = c.take<int32_t>((size_t)rows * k);
  w.top = c.take<int32_t>(k ? rows : 0);
  w.live = c.take<int32_t>(k ? rows : 0);
  w.bytes = c.used + 256;
  return w;
}

// Classes per piece of the backward pass: the piece's dz takes 2 bytes per row and class; at most PIECE_BYTES, but not so few classes that
// the products become short (4096).  Pieces are of nearly equal size.  Fewer pieces are faster, as each one adds to the sums of dh in memory
// and starts four kernels (16384 rows x 50257 x 2048: 10.2 ms in 2 pieces, 10.7 in 4, 12.8 in 13).
constexpr long long PIECE_BYTES = 1ll << 30;
static int piece_classes(int rows, int vocab) {
  long long most = PIECE_BYTES / (2 * pad_rows(rows));
  most = most < 4096 ? 4096 : most;
  const long long whole = (vocab + BN - 1) / BN;
  const long long most_tiles = most / BN;
  const long long pieces = (whole + most_tiles - 1) / most_tiles;
  return (int)((whole + pieces - 1) / pieces * BN);
}

struct BwdWs {
  uint16_t* packed;
  int32_t* origin;
  float* lse2;
  int32_t* tgt;
  float* tdiff;
  uint16_t* dz;
  float* acc;
  float* slots;
  int piece;
  size_t bytes;
};
static BwdWs bwd_ws(void* ws, int rows, int vocab, int width) {
  Carver c(ws);
  BwdWs w;
  w.piece = piece_classes(rows, vocab);
  w.packed = c.take<uint16_t>((size_t)pad_rows(rows) * pad_width(width));
  w.origin = c.take<int32_t>(rows);
  w.lse2 = c.take<float>(pad_rows(rows));
  w.tgt = c.take<int32_t>(rows);
  w.tdiff = c.take<float>(rows);
  w.dz = c.take<uint16_t>((size_t)pad_rows(rows) * w.piece);
  w.acc = c.take<float>(w.piece < vocab ? (size_t)pad_rows(rows) * pad_cols(width) : 0);
  const bool split = (w.piece < vocab ? w.piece : vocab) > SPLIT_MIN_KB * BK || rows > SPLIT_MIN_KB * BK;
  w.slots = c.take<float>(split ? (size_t)2 * sm_count() * BM * BN : 0);   // two tiles' parts per worker
  w.bytes = c.used + 256;
  return w;
}

static int check_head(const char* fn, const void* hidden, long long ldh, const void* weight, long long ldw, int rows, int vocab, int width,
                      int dtype, const int32_t* status) {
  LANCET_REQUIRE(dtype == LANCET_BF16 || dtype == LANCET_F16, LANCET_ERR_UNSUPPORTED,
                 "%s: hidden rows and weight must be bfloat16 or float16 (dtype code %d)", fn, dtype);
  LANCET_REQUIRE(rows >= 0 && rows <= (1 << 26) && vocab >= 1 && vocab <= (1 << 26) && width >= 1 && width <= (1 << 20), LANCET_ERR_INVALID,
                 "%s: bad sizes rows=%d vocab=%d width=%d", fn, rows, vocab, width);
  LANCET_REQUIRE(ldh >= width && ldw >= width, LANCET_ERR_INVALID, "%s: row strides %lld / %lld below the width %d", fn, ldh, ldw, width);
  LANCET_REQUIRE(weight && status && (rows == 0 || hidden), LANCET_ERR_NULL, "%s: null pointer argument", fn);
  LANCET_REQUIRE(aligned(weight, 16) && ldw % 8 == 0, LANCET_ERR_INVALID,
                 "%s: the weight's rows must start on 16-byte boundaries (row stride %lld)", fn, ldw);
  LANCET_REQUIRE(aligned(hidden, 2), LANCET_ERR_INVALID, "%s: hidden is not aligned to its type", fn);
  return LANCET_OK;
}
static int check_teacher(const char* fn, int k, float temperature) {
  LANCET_REQUIRE(k >= 1 && k <= kMaxTop, LANCET_ERR_INVALID, "%s: k=%d top entries (1 to %d)", fn, k, kMaxTop);
  LANCET_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, LANCET_ERR_INVALID, "%s: temperature %g outside [0.001, 1000]", fn,
                 (double)temperature);
  return LANCET_OK;
}

struct FwdArgs {
  const void* hidden;
  long long ldh;
  const void* weight;
  long long ldw;
  const long long* target;
  const void* values;
  int vdtype;
  const long long* indices;
  int k;
  float inv_t;
  int rows, vocab, width, dtype;
  float *loss_rows, *lse_rows, *diff;
  int32_t* pos;
  float *mean, *inv_live;
  void* ws;
  size_t ws_bytes;
  int32_t* status;
};

template <typename T, bool TEACHER>
static int finish_launch(const FwdArgs& a, const FwdWs& w, int n_part, cudaStream_t st) {
  const FinishArgs f = {w.part, pad_rows(a.rows), n_part, a.pos + a.rows, w.origin, w.packed, pad_width(a.width), a.weight, a.ldw, a.width,
                        w.tgt, w.zt, w.idx, w.q, w.cw, a.k, a.inv_t, a.loss_rows, a.lse_rows, a.diff, w.block_sums, w.done, a.mean, a.inv_live};
  auto go = [&](auto kernel, int rows_per_block) {
    const size_t smem = TEACHER ? (size_t)rows_per_block * a.k * sizeof(float) : 0;   // at most 16 KB
    launch_chained(kernel, dim3((a.rows + rows_per_block - 1) / rows_per_block), dim3(kFinishThreads), smem, st, f);
    return launch_status("finish_rows_kernel");
  };
  // 8 rows a block read the partial sums in whole sectors; with few rows, or many entries of teachers, more blocks (captured forward passes, 1 / 8
  // rows a block: targets at 32000 x 256 512 rows 21.5 / 22.3 us, 1024 rows 30.7 / 29.3; teachers at 50257 x 1024 k = 16 640 rows 82 / 88, 1024
  // rows 108 / 104; k = 64 1536 rows 171 / 194, 2972 rows 322 / 299; k = 256 4096 rows 717 / 844, at 32000 x 256 6000 rows 356 / 337)
  constexpr int ENTRY_ROWS = 20;
  if (a.rows > 512 + (TEACHER ? ENTRY_ROWS * a.k : 0)) return go(finish_rows_kernel<T, 8, TEACHER>, 8);
  return go(finish_rows_kernel<T, 1, TEACHER>, 1);
}
template <typename T>
static int finish_launch(const FwdArgs& a, const FwdWs& w, int n_part, cudaStream_t st) {
  return a.target ? finish_launch<T, false>(a, w, n_part, st) : finish_launch<T, true>(a, w, n_part, st);
}

static int linear_fwd(const char* fn, const FwdArgs& a, cudaStream_t st) {
  if (a.rows == 0) return launch_mean(nullptr, nullptr, 0, a.mean, a.inv_live, st);
  const FwdWs w = fwd_ws(a.ws, a.rows, a.vocab, a.width, a.target ? 0 : a.k);
  LANCET_REQUIRE(a.ws && aligned(a.ws, 256) && a.ws_bytes >= w.bytes, LANCET_ERR_INVALID,
                 "%s: workspace missing, not aligned to 256 bytes or smaller than %zu bytes", fn, w.bytes);
  if (!a.target) {
    launch_chained(teacher_kernel, dim3((a.rows + kTeacherWarps - 1) / kTeacherWarps), dim3(32 * kTeacherWarps), 0, st, a.values, a.vdtype,
                   a.indices, a.rows, a.k, a.inv_t, a.vocab, w.q, w.cw, w.idx, w.top, w.live);
    if (int rc = launch_status("teacher_kernel")) return rc;
  }
  int blocks = (a.rows + 7) / 8;
  blocks = blocks > 4 * sm_count() ? 4 * sm_count() : blocks;
  launch_chained(pack_rows_kernel, dim3(blocks), dim3(kRowThreads), 0, st, static_cast<const uint16_t*>(a.hidden), a.ldh, a.target,
                 static_cast<const int32_t*>(a.target ? nullptr : w.live), static_cast<const int32_t*>(w.top), a.rows, a.vocab, a.width, w.packed, pad_width(a.width), w.origin,
                 w.tgt, a.pos, a.loss_rows, a.lse_rows, w.done);
  if (int rc = launch_status("pack_rows_kernel")) return rc;
  const bool paired = paired_for(a.rows);
  CUtensorMap tmA, tmB;
  if (int rc = make_map(&tmA, w.packed, pad_rows(a.rows), a.width, pad_width(a.width), BM, a.dtype)) return rc;
  if (int rc = make_map(&tmB, a.weight, a.vocab, a.width, a.ldw, paired ? BN / 2 : BN, a.dtype)) return rc;
  Params p = {};
  p.count = a.pos + a.rows;
  p.classes = a.vocab;
  p.width = a.width;
  p.status = a.status;
  p.c = a.inv_t * kLog2e;
  p.part = w.part;
  p.part_ld = pad_rows(a.rows);
  p.tgt = w.tgt;
  p.zt = w.zt;
  int rc = a.dtype == LANCET_BF16 ? launch_product<__nv_bfloat16, FORM_Z, EPI_LSE>(tmA, tmB, tmA, p, a.rows, a.vocab, a.width, paired, st)
                                  : launch_product<__half, FORM_Z, EPI_LSE>(tmA, tmB, tmA, p, a.rows, a.vocab, a.width, paired, st);
  if (rc) return rc;
  const int n_part = 2 * ((a.vocab + BN - 1) / BN);
  return a.dtype == LANCET_BF16 ? finish_launch<__nv_bfloat16>(a, w, n_part, st) : finish_launch<__half>(a, w, n_part, st);
}

struct BwdArgs {
  const void* hidden;
  long long ldh;
  const void* weight;
  long long ldw;
  const long long* target;
  const float* loss_rows;
  const long long* indices;
  const float* diff;
  int k;
  float inv_t;
  const float* lse_rows;
  const int32_t* pos;
  int rows, vocab, weight_rows, width, dtype;
  const float* grad_out;
  const float* inv_live;
  float scale;
  void *dhidden, *dweight;
  void* ws;
  size_t ws_bytes;
  int32_t* status;
};

template <typename T>
static int linear_bwd_t(const BwdArgs& a, const BwdWs& w, cudaStream_t st) {
  // dz is kept in 16 bits.  In float16 it carries a factor of 2^14 (its values are within [-1, 1]): probabilities keep 11 bits down to 2^-28
  // (2^-14 without it) and steps of 2^-38 below (2^-24); the factor leaves again in the products' float32 results.
  const float shift = a.dtype == LANCET_F16 ? 14.f : 0.f;
  const float unit = a.dtype == LANCET_F16 ? 16384.f : 1.f;
  int blocks = (a.rows + 7) / 8;
  blocks = blocks > 4 * sm_count() ? 4 * sm_count() : (blocks < 8 ? 8 : blocks);   // the zero rows want some warps even for one row
  launch_chained(repack_rows_kernel, dim3(blocks), dim3(kRowThreads), 0, st, static_cast<const uint16_t*>(a.hidden), a.ldh, a.pos, a.lse_rows,
                 a.target, a.loss_rows, unit, a.rows, a.width, w.packed, pad_width(a.width), w.origin, w.lse2, w.tgt, w.tdiff,
                 static_cast<uint16_t*>(a.dhidden));
  if (int rc = launch_status("repack_rows_kernel")) return rc;
  const bool paired = paired_for(a.rows);
  const long long padded = pad_rows(a.rows);
  Params p = {};
  p.count = a.pos + a.rows;
  p.width = a.width;
  p.status = a.status;
  p.c = a.inv_t * kLog2e;
  p.lse2 = w.lse2;
  p.shift = shift;
  p.tgt = a.target ? w.tgt : nullptr;
  p.tdiff = w.tdiff;
  p.grad_out = a.grad_out;
  p.inv_live = a.inv_live;
  p.slots = w.slots;
  p.scale = a.scale / (a.inv_t * unit);
  CUtensorMap hK, wK, dzK, wMN, dzMN, hMN, dzOut, dwOut;
  if (int rc = make_map(&hK, w.packed, padded, a.width, pad_width(a.width), BM, a.dtype)) return rc;
  if (int rc = make_map(&wK, a.weight, a.vocab, a.width, a.ldw, paired ? BN / 2 : BN, a.dtype)) return rc;
  if (int rc = make_map(&dzK, w.dz, padded, w.piece, w.piece, BM, a.dtype)) return rc;
  if (int rc = make_map(&wMN, a.weight, a.vocab, a.width, a.ldw, 64, a.dtype)) return rc;
  if (int rc = make_map(&dzMN, w.dz, padded, w.piece, w.piece, 64, a.dtype)) return rc;
  if (int rc = make_map(&dzOut, w.dz, padded, w.piece, w.piece, OUT_ROWS, a.dtype)) return rc;
  const bool boxes = a.dweight && a.width % 8 == 0 && aligned(a.dweight, 16);
  dwOut = dzOut;
  if (boxes)   // rows behind the vocabulary are no part of it
    if (int rc = make_map(&dwOut, a.dweight, a.vocab, a.width, a.width, OUT_ROWS, a.dtype)) return rc;
  if (int rc = make_map(&hMN, w.packed, padded, a.width, pad_width(a.width), 64, a.dtype)) return rc;
  for (int v0 = 0; v0 < a.vocab; v0 += w.piece) {
    const int classes = a.vocab - v0 < w.piece ? a.vocab - v0 : w.piece;
    const bool last = v0 + classes == a.vocab;
    p.class0 = v0;
    p.classes = classes;
    if (int rc = launch_product<T, FORM_Z, EPI_PROB>(hK, wK, dzOut, p, a.rows, classes, a.width, paired, st)) return rc;
    if (!a.target) {
      const long long entries = (long long)a.rows * a.k;
      launch_chained(place_targets_kernel<T>, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, st, static_cast<const int32_t*>(p.count),
                     static_cast<const int32_t*>(w.origin), a.indices, a.diff, a.k, v0, classes, unit, reinterpret_cast<T*>(w.dz),
                     (long long)w.piece);
      if (int rc = launch_status("place_targets_kernel")) return rc;
    }
    Params ph = p;
    ph.out = a.dhidden;
    ph.row_map = w.origin;
    if (w.piece < a.vocab) {
      ph.acc = w.acc;
      ph.acc_ld = pad_cols(a.width);
      ph.acc_in = v0 > 0;
      ph.acc_out = !last;
    }
    if (a.dhidden)
      if (int rc = launch_product<T, FORM_DH, EPI_OUT>(dzK, wMN, dzK, ph, a.rows, a.width, classes, paired, st)) return rc;
    if (!a.dweight) continue;
    Params pw = p;
    pw.out = a.dweight;
    pw.boxes = boxes;
    if (int rc = launch_product<T, FORM_DW, EPI_OUT>(dzMN, hMN, dwOut, pw, classes, a.width, a.rows, paired_for(classes), st)) return rc;
  }
  return LANCET_OK;
}

static int linear_bwd(const char* fn, const BwdArgs& a, cudaStream_t st) {
  LANCET_REQUIRE(a.weight_rows >= a.vocab, LANCET_ERR_INVALID, "%s: %d weight rows for %d classes", fn, a.weight_rows, a.vocab);
  LANCET_REQUIRE(a.rows == 0 || (a.lse_rows && a.pos), LANCET_ERR_NULL, "%s: null pointer argument", fn);
  LANCET_REQUIRE(aligned(a.dhidden, 2) && aligned(a.dweight, 2), LANCET_ERR_INVALID, "%s: outputs are not aligned to their type", fn);
  const bool work = a.rows > 0 && (a.dhidden || a.dweight);
  const BwdWs w = bwd_ws(a.ws, a.rows, a.vocab, a.width);
  if (work)
    LANCET_REQUIRE(a.ws && aligned(a.ws, 256) && a.ws_bytes >= w.bytes, LANCET_ERR_INVALID,
                   "%s: workspace missing, not aligned to 256 bytes or smaller than %zu bytes", fn, w.bytes);
  uint16_t* dw = static_cast<uint16_t*>(a.dweight);
  const int first = a.rows == 0 ? 0 : a.vocab;   // rows behind the vocabulary have no gradient
  if (dw && first < a.weight_rows)
    LANCET_CUDA(cudaMemsetAsync(dw + (size_t)first * a.width, 0, (size_t)(a.weight_rows - first) * a.width * 2, st));
  if (!work) return LANCET_OK;
  return a.dtype == LANCET_BF16 ? linear_bwd_t<__nv_bfloat16>(a, w, st) : linear_bwd_t<__half>(a, w, st);
}

}  // namespace head
}  // namespace lancet

extern "C" {
using namespace lancet;

int lancet_copy_rows(const void* src, long long lds, void* dst, long long ldd, int rows, int width, lancet_stream_t stream) {
  LANCET_REQUIRE(rows >= 0 && rows <= head::kMostSize && width >= 1 && width <= head::kMostSize && lds >= width && ldd >= width && ldd % 8 == 0,
                 LANCET_ERR_INVALID,
                 "lancet_copy_rows: bad rows=%d, width=%d or row strides %lld / %lld", rows, width, lds, ldd);
  if (rows == 0) return LANCET_OK;
  LANCET_REQUIRE(src && dst, LANCET_ERR_NULL, "lancet_copy_rows: null pointer argument");
  LANCET_REQUIRE(aligned(src, 2) && aligned(dst, 16), LANCET_ERR_INVALID, "lancet_copy_rows: src must be 2-byte, dst 16-byte aligned");
  int blocks = (rows + 7) / 8;
  blocks = blocks > 8 * sm_count() ? 8 * sm_count() : blocks;
  launch_chained(head::copy_rows_kernel, dim3(blocks), dim3(head::kRowThreads), 0, static_cast<cudaStream_t>(stream),
                 static_cast<const uint16_t*>(src), lds, static_cast<uint16_t*>(dst), ldd, rows, width);
  return launch_status("copy_rows_kernel");
}

size_t lancet_linear_loss_fwd_workspace_bytes(int rows, int vocab, int width, int k) {
  if (rows < 0 || vocab < 1 || width < 1 || k < 0) return 0;
  return head::fwd_ws(nullptr, rows, vocab, width, k).bytes;
}
size_t lancet_linear_loss_bwd_workspace_bytes(int rows, int vocab, int width) {
  if (rows < 0 || vocab < 1 || width < 1) return 0;
  return head::bwd_ws(nullptr, rows, vocab, width).bytes;
}

int lancet_linear_xent_fwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, int rows, int vocab,
                           int width, int dtype, float* loss_rows, float* lse_rows, int32_t* pos, float* mean, float* inv_live, void* ws, size_t ws_bytes,
                           int32_t* status, lancet_stream_t stream) {
  const char* fn = "lancet_linear_xent_fwd";
  if (int rc = head::check_head(fn, hidden, ldh, weight, ldw, rows, vocab, width, dtype, status)) return rc;
  LANCET_REQUIRE(mean && inv_live && (rows == 0 || (target && loss_rows && lse_rows && pos)), LANCET_ERR_NULL, "%s: null pointer argument", fn);
  const head::FwdArgs a = {hidden, ldh, weight, ldw, target, nullptr, 0, nullptr, 1, 1.f, rows, vocab, width, dtype, loss_rows, lse_rows,
                           nullptr, pos, mean, inv_live, ws, ws_bytes, status};
  return head::linear_fwd(fn, a, static_cast<cudaStream_t>(stream));
}

int lancet_linear_xent_bwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target,
                           const float* loss_rows, const float* lse_rows, const int32_t* pos, int rows, int vocab, int weight_rows, int width,
                           int dtype, const float* grad_out, const float* inv_live, float scale, void* dhidden, void* dweight, void* ws,
                           size_t ws_bytes, int32_t* status, lancet_stream_t stream) {
  const char* fn = "lancet_linear_xent_bwd";
  if (int rc = head::check_head(fn, hidden, ldh, weight, ldw, rows, vocab, width, dtype, status)) return rc;
  LANCET_REQUIRE(rows == 0 || (target && loss_rows), LANCET_ERR_NULL, "%s: null pointer argument", fn);
  const head::BwdArgs a = {hidden, ldh, weight, ldw, target, loss_rows, nullptr, nullptr, 1, 1.f, lse_rows, pos, rows, vocab, weight_rows,
                           width, dtype, grad_out, inv_live, scale, dhidden, dweight, ws, ws_bytes, status};
  return head::linear_bwd(fn, a, static_cast<cudaStream_t>(stream));
}

int lancet_linear_distill_fwd(const void* hidden, long long ldh, const void* weight, long long ldw, const void* top_values, int values_dtype,
                              const long long* top_indices, int k, float temperature, int rows, int vocab, int width, int dtype,
                              float* loss_rows, float* lse_rows, float* diff, int32_t* pos, float* mean, float* inv_live, void* ws, size_t ws_bytes,
                              int32_t* status, lancet_stream_t stream) {
  const char* fn = "lancet_linear_distill_fwd";
  if (int rc = head::check_head(fn, hidden, ldh, weight, ldw, rows, vocab, width, dtype, status)) return rc;
  if (int rc = head::check_teacher(fn, k, temperature)) return rc;
  LANCET_REQUIRE(valid_dtype(values_dtype), LANCET_ERR_INVALID, "%s: unknown dtype code %d of the values", fn, values_dtype);
  LANCET_REQUIRE(mean && inv_live && (rows == 0 || (top_values && top_indices && loss_rows && lse_rows && diff && pos)), LANCET_ERR_NULL,
                 "%s: null pointer argument", fn);
  const head::FwdArgs a = {hidden, ldh, weight, ldw, nullptr, top_values, values_dtype, top_indices, k, 1.0f / temperature, rows, vocab, width,
                           dtype, loss_rows, lse_rows, diff, pos, mean, inv_live, ws, ws_bytes, status};
  return head::linear_fwd(fn, a, static_cast<cudaStream_t>(stream));
}

int lancet_linear_distill_bwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* top_indices,
                              const float* diff, int k, float temperature, const float* lse_rows, const int32_t* pos, int rows, int vocab,
                              int weight_rows, int width, int dtype, const float* grad_out, const float* inv_live, float scale, void* dhidden,
                              void* dweight, void* ws, size_t ws_bytes, int32_t* status, lancet_stream_t stream) {
  const char* fn = "lancet_linear_distill_bwd";
  if (int rc = head::check_head(fn, hidden, ldh, weight, ldw, rows, vocab, width, dtype, status)) return rc;
  if (int rc = head::check_teacher(fn, k, temperature)) return rc;
  LANCET_REQUIRE(rows == 0 || (top_indices && diff), LANCET_ERR_NULL, "%s: null pointer argument", fn);
  const head::BwdArgs a = {hidden, ldh, weight, ldw, nullptr, nullptr, top_indices, diff, k, 1.0f / temperature, lse_rows, pos, rows, vocab,
                           weight_rows, width, dtype, grad_out, inv_live, scale, dhidden, dweight, ws, ws_bytes, status};
  return head::linear_bwd(fn, a, static_cast<cudaStream_t>(stream));
}
}
