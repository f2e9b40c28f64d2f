// Product of 8-bit rows with 8-bit weights: out[m, n] = sa[m] * sw[n] * sum_k a[m, k] * w[n, k], a [M, K] and w [N, K] in e4m3, scales fp32,
// sums fp32, bf16 or fp32 output. Both operands go to the tensor cores as they lie in memory; the scales, one a row and one a column, are
// applied to the finished sums. Three kernels by the number of rows:
//   up to 8 rows, and up to 16 where the matrix is small    a stream of the weights through the fragments of mma.sync (no shared memory on the way)
//   up to 256        tcgen05 the other way round, up to 256 rows of w a tile, its k range cut over a cluster
//   more, and from a few rows on where an estimate says it is sooner done    tcgen05, pairs of CTAs on tiles of 256 rows by 256, 128 or 64 columns
// Rows that do not start on 16-byte boundaries go to gemm_quant.cu instead. The bf16 siblings are gemm_skinny.cu, gemm_rows.cu and gemm_tc05.cu;
// the reference sends every product to cuBLAS (src/source/op/kernels/cuda/matmul_kernel.cu:128-150) and has no 8-bit form.
//
// Launched as a programmatic dependent, a kernel may start while the kernels before it still write its operands, the weights too when they have
// just been quantised. So before the wait for them nothing is read; w is only asked into L2 (a hint that keeps no value anywhere else).
#include "tma_common.cuh"
#include "quant_common.cuh"

typedef __nv_bfloat16 bf16;
typedef unsigned char u8;

// Instruction descriptor: e4m3 x e4m3 -> fp32, M x N tile, both operands K-major.
__host__ __device__ constexpr unsigned q8_idesc(int M, int N) { return (1u << 4) | ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24); }

__device__ __forceinline__ void q8_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void q8_mma_pair(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// After a wait that ran out: the copies still under way are waited for (with a limit again) before the block's shared memory goes.
// `issued` k steps have been asked for in all.
__device__ __forceinline__ void drain_copies(uint64_t* full, int stages, int issued) {
  for (int i = issued > stages ? issued - stages : 0; i < issued; ++i) mbar_wait(&full[i % stages], (unsigned)((i / stages) & 1));
}

static int encode_u8_2d(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, unsigned box_rows) {
  SiEncodeTiledFn fn = si_encode_fn();
  if (!fn) return -3;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

// ---- many rows ------------------------------------------------------------------------------------------
// The pipeline of gemm_tc05.cu's pair kernel with e4m3 operands: boxes of 128 entries (128 bytes a row, the swizzle's span), four instructions of
// K = 32 each. A k step is one box where the tile has 256 columns, else two: a wait, a commit and the loop cost some 430 clocks a step, which the instructions
// of narrow tiles do not fill (256 x 4,096 x 14,336, 64 columns: 33.7 us with one box, 23.9 with two; 2,048 x 6,144 x 4,096, 256 columns: 39 and 45). Two CTAs (a cluster) take a tile of 256 x BN: each fetches its 128 rows of a and BN / 2 of w a step, the leader issues
// over both CTAs' shared memory, each CTA stores its 128 rows. Two accumulators in tensor memory: a tile is stored while the next one runs.
template <int STAGES, typename TO, int BN, int BK>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(192, 1)
gemm_q8_pair_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap, const float* sa,
                    const float* sw, TO* __restrict__ out, long long ldo, int M, int N, int K, int* status, int trigger) {
  constexpr int BM = 128, BOXES = BK / 128;               // boxes of 128 entries a step
  constexpr int CW = BN < 128 ? BN : 128;                // columns that an epilogue thread holds at once
  constexpr int A_BYTES = BM * BK, B_BYTES = (BN / 2) * BK;
  extern __shared__ u8 smem_dyn[];
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
  __shared__ unsigned tmem_slot;
  u8* As = reinterpret_cast<u8*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  u8* Bs = As + STAGES * A_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = cluster_cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int m_tiles = (M + 2 * BM - 1) / (2 * BM), n_tiles = (N + BN - 1) / BN;
  const int tiles = m_tiles * n_tiles, nk = (K + BK - 1) / BK;
  if (trigger) pdl_trigger();                             // one block an SM: the next kernel's blocks take no block's place
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
#pragma unroll
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 8); }   // 4 epilogue warps of each CTA
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) tmem_alloc_pair(&tmem_slot, 2 * BN);
  tc05_fence_before_sync();
  cluster_sync_all();
  tc05_fence_after_sync();
  const unsigned tmem = tmem_slot;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = 0; kb < BOXES * nk && kb < BOXES * STAGES; ++kb) tma_prefetch_2d(&bmap, kb * 128, (pair / m_tiles) * BN + (int)rank * (BN / 2));
      pdl_wait();
      int it = 0, s = 0;
      unsigned phase = 1;                                // a stage's first use needs no wait
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        const int m0 = (tile % m_tiles) * 2 * BM + (int)rank * BM, n0 = (tile / m_tiles) * BN + (int)rank * (BN / 2);
        for (int kb = 0; kb < nk; ++kb, ++it) {
          if (it >= STAGES && !mbar_wait(&empty_bar[s], phase)) {
            set_status(status, SI_WAIT_LIMIT);
            ok = false;
            break;
          }
          const unsigned bar = cluster_map_u32(&full_bar[s], 0);
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * (A_BYTES + B_BYTES));
#pragma unroll
          for (int j = 0; j < BOXES; ++j) {
            tma_load_2d_pair(Bs + s * B_BYTES + j * (B_BYTES / BOXES), &bmap, bar, kb * BK + j * 128, n0);
            tma_load_2d_pair(As + s * A_BYTES + j * (A_BYTES / BOXES), &amap, bar, kb * BK + j * 128, m0);
          }
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
      }
      if (!ok && rank == 0) drain_copies(full_bar, STAGES, it);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr unsigned idesc = q8_idesc(2 * BM, BN);
      const unsigned long long ad0 = umma_desc_sw128(As, 16, 1024), bd0 = umma_desc_sw128(Bs, 16, 1024);
      int s = 0, local = 0;
      unsigned phase = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs, ++local) {
        const int buf = local & 1;
        if (local >= 2) ok = mbar_wait_warp(&acc_empty[buf], (unsigned)(((local >> 1) - 1) & 1));
        if (!ok) break;
        tc05_fence_after_sync();
        const unsigned acc = tmem + buf * BN;
        for (int kb = 0; kb < nk; ++kb) {
          ok = mbar_wait_warp(&full_bar[s], phase);
          if (!ok) break;
          tc05_fence_after_sync();
          const unsigned long long ad = ad0 + (unsigned)s * (A_BYTES / 16), bd = bd0 + (unsigned)s * (B_BYTES / 16);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              q8_mma_pair(acc, ad + (k >> 2) * (A_BYTES / BOXES / 16) + 2 * (k & 3), bd + (k >> 2) * (B_BYTES / BOXES / 16) + 2 * (k & 3), idesc, (kb | k) != 0 ? 1u : 0u);
            tc05_commit_pair(&empty_bar[s], 3);
            if (kb == nk - 1) tc05_commit_pair(&acc_full[buf], 3);
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
    }
  } else {
    pdl_wait();
    const int q = warp & 3;
    const bool vec = ldo % (16 / (int)sizeof(TO)) == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)sw % 16 == 0;
    int local = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++local) {
      const int buf = local & 1;
      const int row = (tile % m_tiles) * 2 * BM + (int)rank * BM + q * 32 + lane, n0 = (tile / m_tiles) * BN;
      const float rs = row < M ? sa[row] : 0.f;
      const bool plain = q8_plain(rs, q8_range(sw, n0, min(n0 + BN, N)));
      if (!mbar_wait_warp(&acc_full[buf], (unsigned)((local >> 1) & 1))) {
        if (lane == 0) set_status(status, SI_WAIT_LIMIT);
        break;
      }
      tc05_fence_after_sync();
      const unsigned src = tmem + ((unsigned)(q * 32) << 16) + (unsigned)(buf * BN);
#pragma unroll 1
      for (int h = 0; h < BN / CW; ++h) {
        float v[CW / 32][32];
        __syncwarp();                            // an aligned load: not every lane stored in the turn before
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) tmem_ld_32x32_issue(src + h * CW + c * 32, v[c]);
        tmem_ld_wait();
        if (h == BN / CW - 1) {                  // in registers: the leader's issuer may have the accumulator back
          tc05_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_map_u32(&acc_empty[buf], 0));
        }
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) {
          const int n = n0 + h * CW + c * 32;
          if (row < M && n < N) {
            TO* dst = out + (size_t)row * ldo + n;
            if (vec && n + 32 <= N) {
              if (plain) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float4 s4 = reinterpret_cast<const float4*>(sw + n)[i];
                  v[c][4 * i] *= rs * s4.x; v[c][4 * i + 1] *= rs * s4.y; v[c][4 * i + 2] *= rs * s4.z; v[c][4 * i + 3] *= rs * s4.w;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[c][i] = q8_scaled_wide(v[c][i], rs, sw[n + i]);
              }
              if constexpr (sizeof(TO) == 4) {
#pragma unroll
                for (int i = 0; i < 8; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(v[c][4 * i], v[c][4 * i + 1], v[c][4 * i + 2], v[c][4 * i + 3]);
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  uint4 raw;
                  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
                  for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(v[c][8 * i + 2 * j], v[c][8 * i + 2 * j + 1]);
                  reinterpret_cast<uint4*>(dst)[i] = raw;
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) if (n + i < N) dst[i] = from_f32<TO>(plain ? v[c][i] * (rs * sw[n + i]) : q8_scaled_wide(v[c][i], rs, sw[n + i]));
            }
          }
        }
      }
    }
  }
  tc05_fence_before_sync();
  cluster_sync_all();                                     // no CTA frees tensor memory the other one's instructions use
  if (warp == 1) tmem_dealloc_pair(tmem, 2 * BN);
}

// Columns of a pair's tile: those for which the busiest pair is done first. In clocks: 256 entries of k take 1,120, 750 or 630 with tiles of 256, 128 and
// 64 columns, what comes before and after them 15,800, 10,560 and 9,300 once. us with 64, 128, 256: 512 x 4,096 x 14,336 42, 28, 41; 512 x 2,048 x
// 2,048 7.3, 8.1, 12.4; 1,024 x 6,144 x 4,096 37, 24, 28; 1,024 x 4,096 x 14,336 79, 50, 44; 2,048 x 6,144 x 4,096 65, 43, 40.
static int q8_pair_columns(int M, int N, int K, long long* cost) {
  const long long slots = si_sm_count() / 2, m_tiles = (M + 255) / 256, nk = (K + 255) / 256;
  int best = 256;
  *cost = -1;
  for (int bn = 256; bn >= 64; bn /= 2) {
    const long long rounds = (m_tiles * ((N + bn - 1) / bn) + slots - 1) / slots;
    const long long c = rounds * nk * (bn == 256 ? 1120 : bn == 128 ? 750 : 630) + (bn == 256 ? 15800 : bn == 128 ? 10560 : 9300);
    if (*cost < 0 || c < *cost) { *cost = c; best = bn; }
  }
  return best;
}

struct Q8Call {
  const void* a; long long lda; const float* sa; const void* w; long long ldw; const float* sw;
  void* out; long long ldo; int M, N, K; int* status; cudaStream_t stream;
};

template <typename TO, int BN>
static int q8_pair(const Q8Call& c) {
  constexpr int BK = BN == 256 ? 128 : 256, STAGES = BN == 256 ? 6 : BN == 128 ? 4 : 5;
  const size_t smem = (size_t)STAGES * (128 + BN / 2) * BK + 1024;
  auto k = gemm_q8_pair_kernel<STAGES, TO, BN, BK>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  CUtensorMap am, bm;
  int rc = encode_u8_2d(&am, c.a, c.M, c.K, c.lda, 128);
  if (!rc) rc = encode_u8_2d(&bm, c.w, c.N, c.K, c.ldw, BN / 2);
  if (rc) return rc;
  const long long tiles = (long long)((c.M + 255) / 256) * ((c.N + BN - 1) / BN), slots = si_sm_count() / 2;
  if (tiles > 0x3fffffffLL || slots < 1) return -2;
  const long long blocks = 2 * (tiles < slots ? tiles : slots);
  si_launch(k, dim3((unsigned)blocks), dim3(192), smem, c.stream, am, bm, c.sa, c.sw, (TO*)c.out, c.ldo, c.M, c.N, c.K, c.status,
            si_pdl_trigger_mode(blocks, si_sm_count()));
  return si_last_error();
}

// ---- 17 to 256 rows ----------------------------------------------------------------------------------------------
// One pass over the weights, the product taken the other way round: `h` rows of w are the M of the instruction (one or two of 128 rows; what lies
// in shared memory behind row h - 1 makes sums that nobody reads), the rows of a, padded to 16, its N, and the accumulator holds out
// transposed. One block an SM, a ring of as many stages of [h x 256] of w and [rows x 256] of a as 208 KB hold. What bounds it: a wait, the
// instructions and a commit cost the issuing thread some 430 clocks a step whatever the step's bytes (steps of 128 took 520 in all, so 256 are
// taken), and a block some 3 us to begin, to meet the others and to end. The height h, any multiple of 8 up to 256, is chosen with the cut of k so that the
// SMs share the bytes evenly (q8_rows_shape). The k range of a tile may be cut over the blocks of a cluster: each leaves its sums in its shared
// memory, and block r adds the r-th part of the rows up over all blocks, in their order. us (TB/s of the weights): 61 x 28,672 x 4,096 24.5 (4.8),
// 61 x 4,096 x 14,336 14.2 (4.1), 61 x 6,144 x 4,096 10.0, 128 x 4,096 x 14,336 16.7.
#define Q8_ROWS_MAX 256
#define Q8_ROWS_SMEM (208 * 1024)
#define Q8_ROWS_MAX_STAGES 8
__device__ __forceinline__ float4 ld_cluster_f32x4(unsigned cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
// Stages of a ring: the last stage of w is read up to the instruction's last row, which has to lie in the block's shared memory as well.
__host__ __device__ inline int q8_rows_stages(int h, int mpad) {
  const int n = Q8_ROWS_SMEM / ((h + mpad) * 256);
  return n < Q8_ROWS_MAX_STAGES ? n : Q8_ROWS_MAX_STAGES;
}

template <typename TO>
__global__ void __launch_bounds__(352, 1)
gemm_q8_rows_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap wmap, const float* sa,
                    const float* sw, TO* __restrict__ out, long long ldo, int M, int N, int K, int h, int parts, int* status, int trigger) {
  constexpr int BK = 256;                                  // two boxes of 128 entries: a wait and a commit for eight instructions
  extern __shared__ u8 smem_dyn[];
  __shared__ __align__(8) uint64_t full_bar[Q8_ROWS_MAX_STAGES], empty_bar[Q8_ROWS_MAX_STAGES], acc_full;
  __shared__ unsigned tmem_slot;
  u8* smem = reinterpret_cast<u8*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mpad = (M + 15) & ~15, W_BYTES = h * BK, A_BYTES = mpad * BK, STAGES = q8_rows_stages(h, mpad);
  u8* Ws = smem;
  u8* As = smem + STAGES * W_BYTES;
  float* partial = reinterpret_cast<float*>(smem);         // [mpad][h] once the operands are used up
  const int nk = (K + BK - 1) / BK, halves = h > 128 ? 2 : 1;
  const int part = (int)cluster_cta_rank(), n0 = (int)(blockIdx.x / parts) * h;
  const int k0 = (int)((long long)nk * part / parts), k1 = (int)((long long)nk * (part + 1) / parts), steps = k1 - k0;
  const unsigned acc_cols = mpad <= 32 ? 32 : mpad <= 64 ? 64 : mpad <= 128 ? 128 : 256;
  if (trigger) pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 2); mbar_init(&empty_bar[s], 1); }
    mbar_init(&acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 2) tmem_alloc(&tmem_slot, 2 * acc_cols);
  tc05_fence_before_sync();
  __syncthreads();
  tc05_fence_after_sync();
  const unsigned tmem = tmem_slot;
  bool plain = true;                                       // the scales' products are normal numbers
  // Stages and phases are counted along: a division a step, in the one thread that feeds a pipeline, cost 80 clocks a step.
  if (warp < 2) {                                          // warp 0 fetches w, warp 1 a: each boxes of its own
    if (lane == 0) {
      const CUtensorMap* map = warp == 0 ? &wmap : &amap;
      u8* dst = warp == 0 ? Ws : As;
      const int bytes = warp == 0 ? W_BYTES : A_BYTES, y = warp == 0 ? n0 : 0;
      if (warp == 0)
        for (int i = 0; i < 2 * steps && i < 2 * STAGES; ++i) tma_prefetch_2d(&wmap, k0 * BK + i * 128, n0);
      pdl_wait();
      int s = 0, x = k0 * BK;
      unsigned phase = 1;                                  // a stage's first use needs no wait
      u8* to = dst;
      for (int it = 0; it < steps; ++it) {
        if (it >= STAGES && !mbar_wait(&empty_bar[s], phase)) {
          set_status(status, SI_WAIT_LIMIT);
          drain_copies(full_bar, STAGES, it);
          break;
        }
        mbar_expect_tx(&full_bar[s], (unsigned)bytes);     // both arrive, each with its own bytes
        tma_load_2d(to, map, &full_bar[s], x, y);
        tma_load_2d(to + bytes / 2, map, &full_bar[s], x + 128, y);
        x += BK;
        to += bytes;
        if (++s == STAGES) { s = 0; to = dst; phase ^= 1u; }
      }
    }
  } else if (warp == 2) {
    const unsigned idesc = q8_idesc(128, mpad);
    const unsigned long long wd0 = umma_desc_sw128(Ws, 16, 1024), ad0 = umma_desc_sw128(As, 16, 1024);
    const unsigned w_step = (unsigned)W_BYTES / 16, a_step = (unsigned)A_BYTES / 16;
    unsigned long long wd = wd0, ad = ad0;
    unsigned phase = 0;
    int s = 0;
    bool ok = true;
    for (int it = 0; it < steps; ++it) {
      ok = mbar_wait_warp(&full_bar[s], phase);
      if (!ok) break;
      tc05_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          q8_mma(tmem, wd + (k >> 2) * (w_step / 2) + 2 * (k & 3), ad + (k >> 2) * (a_step / 2) + 2 * (k & 3), idesc, (it | k) != 0 ? 1u : 0u);
        if (halves == 2) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            q8_mma(tmem + acc_cols, wd + 1024 + (k >> 2) * (w_step / 2) + 2 * (k & 3), ad + (k >> 2) * (a_step / 2) + 2 * (k & 3), idesc, (it | k) != 0 ? 1u : 0u);
        }
        tc05_commit(&empty_bar[s]);
        if (it + 1 == steps) tc05_commit(&acc_full);
      }
      __syncwarp();
      wd += w_step;
      ad += a_step;
      if (++s == STAGES) { s = 0; wd = wd0; ad = ad0; phase ^= 1u; }
    }
    if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
  } else {
    pdl_wait();
    const float2 rows = q8_range(sa, 0, M), cols = q8_range(sw, n0, min(n0 + h, N));      // while the product runs
    plain = q8_normal(rows.x * cols.x) && q8_normal(rows.y * cols.y);
  }
  if (warp >= 3 && warp - 3 < 4 * halves) {                 // four warps an accumulator, 32 of its lanes each
    const int acc = (warp - 3) >> 2, c = acc * 128 + (warp & 3) * 32 + lane, n = n0 + c;
    const bool in = c < h && n < N;
    const float cs = in ? sw[n] : 0.f;
    const bool ok = mbar_wait_warp(&acc_full, 0);         // every part has a step at least
    if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
    tc05_fence_after_sync();
    const unsigned src = tmem + ((unsigned)((warp & 3) * 32) << 16) + (unsigned)acc * acc_cols;
#pragma unroll 1
    for (int m0 = 0; m0 < mpad && ok; m0 += 32) {
      float v[32];
      __syncwarp();                                        // an aligned load: not every lane stored in the turn before
      tmem_ld_32x32(src + m0, v);
      if (parts == 1) {
        if (plain) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (m0 + j < M && in) out[(size_t)(m0 + j) * ldo + n] = from_f32<TO>(v[j] * (sa[m0 + j] * cs));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (m0 + j < M && in) out[(size_t)(m0 + j) * ldo + n] = from_f32<TO>(q8_scaled(v[j], sa[m0 + j], cs));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (m0 + j < mpad && c < h) partial[(m0 + j) * h + c] = v[j];
      }
    }
  }
  if (parts > 1) {
    cluster_sync_all();                                   // every block's sums lie in its shared memory
    if (warp >= 3) {
      // four columns a thread, the parts' sums all on their way before the first is used
      const int lo = mpad * part / parts, hi = min(M, mpad * (part + 1) / parts), quads = h / 4;
      const bool vec = ldo % 4 == 0 && (uintptr_t)out % 16 == 0;
      for (int i = (int)threadIdx.x - 96; i < (hi - lo) * quads; i += 256) {
        const int m = lo + i / quads, c4 = (i % quads) * 4, n = n0 + c4;
        const float* at = partial + m * h + c4;
        float4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = c < parts ? ld_cluster_f32x4(cluster_map_u32(at, (unsigned)c)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 1; c < 8; ++c) { v[0].x += v[c].x; v[0].y += v[c].y; v[0].z += v[c].z; v[0].w += v[c].w; }
        const float rs = sa[m];
        const float r[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
        TO* dst = out + (size_t)m * ldo + n;
        if (plain && vec && n + 4 <= N) {
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = r[j] * (rs * sw[n + j]);
          if constexpr (sizeof(TO) == 4) {
            *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
          } else {
            __nv_bfloat162 p[2] = {__floats2bfloat162_rn(y[0], y[1]), __floats2bfloat162_rn(y[2], y[3])};
            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(p);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) if (n + j < N) dst[j] = from_f32<TO>(q8_scaled(r[j], rs, sw[n + j]));
        }
      }
    }
    cluster_sync_all();                                   // no block goes while another one reads its sums
  }
  __syncwarp();
  tc05_fence_before_sync();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, 2 * acc_cols);
}

template <typename TO>
static cudaLaunchConfig_t q8_rows_config(unsigned blocks, int parts, cudaStream_t stream, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(352);
  cfg.dynamicSmemBytes = Q8_ROWS_SMEM + 1024;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = si_pdl_enabled() ? 2 : 1;
  return cfg;
}

// Clusters of `parts` blocks that the device runs at once (the SMs of a cluster lie together, so not every one finds its place), asked
// once per device and size.
template <typename TO>
static int q8_rows_clusters(int parts) {
  static int known[64][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (parts == 1) return si_sm_count();
  if (!known[dev][parts]) {
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = q8_rows_config<TO>((unsigned)parts, parts, 0, attr);
    int n = 0;
    if (cudaFuncSetAttribute(gemm_q8_rows_kernel<TO>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8_ROWS_SMEM + 1024) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, gemm_q8_rows_kernel<TO>, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = 1; }
    known[dev][parts] = n;
  }
  return known[dev][parts];
}

// Height of a tile and blocks that share one: the pair for which the busiest SM is done first. In clocks: a step of 256 takes 850 however few its
// rows are (instructions, a wait, a commit), 400 more for the second instruction row, or, if that is more, its bytes of w at 32 a clock and of a, which
// come from the L2 cache, at 51; a block 6,000 to begin and to end, 2,500 more where a cluster meets, and 50 a row of a to store.
template <typename TO>
static long long q8_rows_shape(int N, int K, int mpad, int* height, int* cut) {
  const int nk = (K + 255) / 256;
  long long least = -1;
  for (int parts = 1; parts <= 8 && parts <= nk; parts *= 2) {
    const int slots = q8_rows_clusters<TO>(parts), steps = (nk + parts - 1) / parts;
    for (int h = 16; h <= 256; h += 8) {
      if (q8_rows_stages(h, mpad) < 2 || (parts > 1 && mpad * h * 4 > Q8_ROWS_SMEM)) break;       // two stages, and the sums that a cluster adds up
      const long long tiles = (N + h - 1) / h, rounds = (tiles + slots - 1) / slots;
      const long long busy = h > 128 ? 1250 : 850, bytes = h * 8 + mpad * 5;
      const long long cost = rounds * (steps * (busy > bytes ? busy : bytes) + (parts > 1 ? 8500 : 6000));
      if (least < 0 || cost < least) { least = cost; *height = h; *cut = parts; }
    }
  }
  return least + 50 * mpad;
}

template <typename TO>
static int q8_rows(const Q8Call& c, int h, int parts) {
  auto k = gemm_q8_rows_kernel<TO>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8_ROWS_SMEM + 1024);
  if (e != cudaSuccess) return (int)e;
  const int mpad = (c.M + 15) & ~15;
  CUtensorMap am, wm;
  int rc = encode_u8_2d(&am, c.a, c.M, c.K, c.lda, (unsigned)mpad);
  if (!rc) rc = encode_u8_2d(&wm, c.w, c.N, c.K, c.ldw, (unsigned)h);
  if (rc) return rc;
  const long long blocks = (long long)((c.N + h - 1) / h) * parts;
  if (blocks > 0x7fffffffLL) return -2;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = q8_rows_config<TO>((unsigned)blocks, parts, c.stream, attr);
  cudaLaunchKernelEx(&cfg, k, am, wm, c.sa, c.sw, (TO*)c.out, c.ldo, c.M, c.N, c.K, h, parts, c.status, si_pdl_trigger_mode(blocks, si_sm_count()));
  return si_last_error();
}

// ---- up to 16 rows -----------------------------------------------------------------------------------------------
// The weights go from global memory straight into the A fragments of mma.sync m16n8k32 (rows of w are the instruction's 16, rows of a its 8),
// 16 bytes a lane and load. Lane (g, t) holds w[n0 + g][k .. k + 16), w[n0 + g + 8][k .. k + 16) and a[g][k .. k + 16), k = 64 c + 16 t: the sum
// does not care in which order k is visited, so the sixteen bytes are fed as the two 4-byte pieces of two instructions, alike for both operands.
// A tile is 16 columns; a block's warps take the 64-wide chunks of k in turn, U of them in flight, and add their sums in warp order.
__device__ __forceinline__ void q8_mma16832(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Loads without a branch: what is not taken becomes zeros. w is read once and kept out of L1, a is shared by all blocks.
__device__ __forceinline__ uint4 q8_ld_w(const u8* p, bool take) {
  uint4 v;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
               "@q ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}\n"
               : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)take) : "memory");
  return v;
}
__device__ __forceinline__ uint4 q8_ld_a(const u8* p, bool take) {
  uint4 v;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
               "@q ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}\n"
               : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)take) : "memory");
  return v;
}

template <int MT, int WARPS, int U, typename TO>
__global__ void __launch_bounds__(WARPS * 32, 512 / (WARPS * 32))
gemm_q8_skinny_kernel(const u8* a, long long lda, const float* sa, const u8* w, long long ldw,
                      const float* sw, TO* __restrict__ out, long long ldo, int M, int N, int K, int tiles, int trigger) {
  __shared__ float red[2][WARPS * MT * 32][4];
  if (trigger) pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rounds = (K + 64 * WARPS * U - 1) / (64 * WARPS * U);
  int tile = blockIdx.x, r = 0;                          // whose loads were asked for last
  uint4 lo[U], hi[U], xb[U][MT];
  auto load = [&]() {
    const u8* w0 = w + (size_t)(tile * 16 + g < N ? tile * 16 + g : 0) * ldw;          // rows beyond N stand for row 0 and are not stored
    const u8* w1 = w + (size_t)(tile * 16 + 8 + g < N ? tile * 16 + 8 + g : 0) * ldw;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (warp + (r * U + u) * WARPS) * 64 + t * 16;
      lo[u] = q8_ld_w(w0 + k, k < K);
      hi[u] = q8_ld_w(w1 + k, k < K);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const bool in = mt * 8 + g < M;
      const u8* ar = a + (size_t)(in ? mt * 8 + g : 0) * lda;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (warp + (r * U + u) * WARPS) * 64 + t * 16;
        xb[u][mt] = q8_ld_a(ar + k, in && k < K);
      }
    }
  };
  {                                                        // the first loads' lines into L2: a lane a row of a chunk
    const int n = tile * 16 + (lane & 15);
    if (n < N)
      for (int u = lane >> 4; u < U; u += 2) {
        const int k = (warp + u * WARPS) * 64;
        if (k < K) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(w + (size_t)n * ldw + k) : "memory");
      }
  }
  pdl_wait();
  load();
  for (int par = 0; tile < tiles; par ^= 1) {
    const int now = tile;
    float acc[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          q8_mma16832(acc[mt], lo[u].x, hi[u].x, lo[u].y, hi[u].y, xb[u][mt].x, xb[u][mt].y);
          q8_mma16832(acc[mt], lo[u].z, hi[u].z, lo[u].w, hi[u].w, xb[u][mt].z, xb[u][mt].w);
        }
      if (++r == rounds) { r = 0; tile += gridDim.x; }
      if (tile < tiles) load();
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      *reinterpret_cast<float4*>(red[par][(warp * MT + mt) * 32 + lane]) = make_float4(acc[mt][0], acc[mt][1], acc[mt][2], acc[mt][3]);
    __syncthreads();
    for (int idx = threadIdx.x; idx < MT * 128; idx += WARPS * 32) {
      const int mt = idx / 128, ln = (idx >> 2) & 31, e = idx & 3;
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < WARPS; ++v) s += red[par][(v * MT + mt) * 32 + ln][e];
      const int n = now * 16 + (ln >> 2) + ((e >> 1) ? 8 : 0), m = mt * 8 + (ln & 3) * 2 + (e & 1);
      if (n < N && m < M) out[(size_t)m * ldo + n] = from_f32<TO>(q8_scaled(s, sa[m], sw[n]));
    }
  }
}

// How many blocks and warps, us (a launch behind a launch, eight rows). Blocks go through the tiles in turn wherever tiles are more than run at
// once: 28,672 x 4,096 24.6 a block a tile, 18.4 so. Four warps a block where K fills no more or all tiles then run at once: 2,048 x 2,048 3.3 with
// eight, 2.9; 6,144 x 4,096 7.0, 6.6. Sixteen where tiles are fewer than SMs and K is more than a round of eight: 2,048 x 8,192 8.8 and 7.0 (16 rows).
// Nine to sixteen rows hold half as many weights in flight; a matrix of more than this goes to the tcgen05 kernel: 4,096 x 4,096 5.9 here, 6.6
// there; 11,264 x 2,048 8.0, 8.0; 6,144 x 4,096 9.3, 8.4; 28,672 x 4,096 25.2, 21.7.
#define Q8_SKINNY_16_MOST (22LL << 20)
template <typename TO>
static int q8_skinny(const Q8Call& c) {
  const long long sms = si_sm_count(), tiles = (c.N + 15) / 16;
  const bool one_round = c.K <= 8 * 8 * 64;
  const int warps = tiles <= sms && !one_round ? 16 : c.M <= 8 && tiles <= 4 * sms && (tiles > 2 * sms || c.K <= 2048) ? 4 : 8;
  const long long slots = 512 / (warps * 32) * sms;
  const dim3 grid((unsigned)(tiles > slots ? slots : tiles)), block(warps * 32);
  const int trig = si_pdl_trigger_mode(grid.x, slots);
#define Q8_SK(MT, WARPS, U) si_launch(gemm_q8_skinny_kernel<MT, WARPS, U, TO>, grid, block, 0, c.stream, (const u8*)c.a, c.lda, c.sa, (const u8*)c.w, \
                                      c.ldw, c.sw, (TO*)c.out, c.ldo, c.M, c.N, c.K, (int)tiles, trig)
  if (c.M > 8) {
    if (warps == 16) Q8_SK(2, 16, 4); else Q8_SK(2, 8, 4);
  } else {
    if (warps == 16) Q8_SK(1, 16, 8); else if (warps == 4) Q8_SK(1, 4, 8); else Q8_SK(1, 8, 8);
  }
#undef Q8_SK
  return si_last_error();
}

// Up to 256 rows the two tcgen05 kernels' costs are compared. us (one CTA and k cut, pairs): 112 x 2,048 x 2,048 9.0, 6.6; 112 x 4,096 x 4,096 9.6, 9.9;
// 136 x 4,096 x 14,336 17.2, 23.5; 136 x 28,672 x 4,096 32.6, 30.2; 176 x 2,048 x 8,192 14.6, 14.8; 256 x 4,096 x 4,096 13.9, 10.1.
template <typename TO>
static int q8_any(const Q8Call& c) {
  if (c.K % 16 == 0 && (c.M <= 8 || (c.M <= 16 && (long long)c.N * c.K <= Q8_SKINNY_16_MOST))) return q8_skinny<TO>(c);
  long long pair_cost;
  const int bn = q8_pair_columns(c.M, c.N, c.K, &pair_cost);
  if (c.M <= Q8_ROWS_MAX) {
    int h = 128, parts = 1;
    const long long cost = q8_rows_shape<TO>(c.N, c.K, (c.M + 15) & ~15, &h, &parts);
    if (cost <= pair_cost) return q8_rows<TO>(c, h, parts);
  }
  switch (bn) {
    case 64: return q8_pair<TO, 64>(c);
    case 128: return q8_pair<TO, 128>(c);
    default: return q8_pair<TO, 256>(c);
  }
}

// 1 when these kernels take operands so laid out (rows that start on 16-byte boundaries, the driver's tensor maps), else gemm_quant.cu does.
SI_EXPORT int si_gemm_q8_ok(const void* a, long long lda, const void* w, long long ldw, int K) {
  return si_encode_fn() != nullptr && ((uintptr_t)a | (uintptr_t)w | (uintptr_t)lda | (uintptr_t)ldw) % 16 == 0 && lda >= K && ldw >= K;
}

// a [M, K] and w [N, K] e4m3, rows `lda` and `ldw` bytes apart (multiples of 16, bases too); sa [M], sw [N] fp32; out [M, N], rows `ldo` entries
// apart, SI_BF16 or SI_F32. Returns 0, a CUDA error code, or -2 (size or layout refused).
static int gemm_q8(const void* a, long long lda, const float* sa, const void* w, long long ldw, const float* sw, void* out,
                         long long ldo, int out_dtype, int M, int N, int K, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 0x3fffffff || !si_gemm_q8_ok(a, lda, w, ldw, K)) return -2;
  Q8Call c;
  c.a = a; c.lda = lda; c.sa = sa; c.w = w; c.ldw = ldw; c.sw = sw; c.out = out; c.ldo = ldo; c.M = M; c.N = N; c.K = K; c.status = status; c.stream = stream;
  return out_dtype == SI_BF16 ? q8_any<bf16>(c) : q8_any<float>(c);
}

// The same with its arguments in one array, in their order (see quant_rows.cu).
SI_EXPORT int si_gemm_q8(const long long* a) {
  return gemm_q8((const void*)a[0], a[1], (const float*)a[2], (const void*)a[3], a[4], (const float*)a[5], (void*)a[6], a[7], (int)a[8], (int)a[9],
                 (int)a[10], (int)a[11], (int*)a[12], (cudaStream_t)a[13]);
}
