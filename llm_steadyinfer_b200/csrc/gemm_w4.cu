// Product of bf16 rows with 4-bit weights: out[m, n] = sum_k x[m, k] * s[n, k / group] * (q[n, k] - z[n, k / group]), sums fp32, bf16 or fp32
// output. q lies in int32 words of eight entries (quant_common.cuh); the weights are widened in registers on their way to the tensor cores and
// never written anywhere in between. Two kernels by the number of rows:
//   up to 16 rows    a stream of the weights through the fragments of mma.sync; q - z is exact in bf16 there and the scale is applied to the
//                    fp32 sum of a group, so no weight is rounded
//   more             tcgen05 the other way round: 128 rows of the weight matrix are the M of the instruction and come to it through tensor memory,
//                    widened and scaled by the warps that own their lanes; a weight times its scale is rounded to bf16 once (2^-8 of it at
//                    most: a scale has eight bits and q - z five, and the instruction takes eight)
// Rows that do not start on 16-byte boundaries go to gemm_quant.cu instead. The reference has no 4-bit form.
//
// Before the wait for the kernels before this one nothing is read, the weights are only asked into L2 (see gemm_q8.cu).
#include "tma_common.cuh"
#include "quant_common.cuh"
#include <stdio.h>

typedef __nv_bfloat16 bf16;

struct W4Call {
  const bf16* x; long long ldx; const unsigned* w; long long ldw; const bf16* scales; const unsigned char* zeros; int group, groups;
  void* out; long long ldo; int M, N, K; int* status; cudaStream_t stream;
};

// ---- up to 16 rows -----------------------------------------------------------------------------------------------
// mma.sync m16n8k16 with 16 rows of the weight matrix as its "m" and up to 8 rows of x as its "n". Lane (g, t) takes WORDS words (8 * WORDS entries)
// of rows n0 + g and n0 + g + 8 at k = 32 * WORDS * c + 8 * WORDS * t, and the same entries of row g of x; a word's four pairs are the k columns of two
// instructions, alike for both operands. A chunk of 32 * WORDS entries lies in one group, so its sums are scaled by the row's number and added
// to the running ones. A tile is 16 columns; a block's warps take the chunks in turn. U chunks of a warp are on their way at a time: as soon as
// one is used, the one U further on, of this tile or the next, is asked for.
__device__ __forceinline__ void w4_mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// WORDS words without a branch: what is not taken becomes zeros. Read once: kept out of L1 where a load takes whole sectors.
template <int WORDS> __device__ __forceinline__ void w4_ld(const unsigned* p, bool take, unsigned (&v)[WORDS]) {
  if constexpr (WORDS == 4)
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
                 "@q ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}\n"
                 : "=&r"(v[0]), "=&r"(v[1]), "=&r"(v[2]), "=&r"(v[3]) : "l"(p), "r"((int)take) : "memory");
  else if constexpr (WORDS == 2)
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %3, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t@q ld.global.v2.u32 {%0,%1}, [%2];\n\t}\n"
                 : "=&r"(v[0]), "=&r"(v[1]) : "l"(p), "r"((int)take) : "memory");
  else
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %2, 0;\n\tmov.u32 %0, 0;\n\t@q ld.global.u32 %0, [%1];\n\t}\n"
                 : "=&r"(v[0]) : "l"(p), "r"((int)take) : "memory");
}
__device__ __forceinline__ uint4 w4_ld_x(const bf16* p, bool take) {
  uint4 v;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
               "@q ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}\n"
               : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)take) : "memory");
  return v;
}

// A scale or a zero point, not by the read-only path: such a load may be moved across the wait for the kernel that writes it.
__device__ __forceinline__ unsigned w4_ld_scale(const bf16* p, bool take) {
  unsigned v;
  asm volatile("{\n\t.reg .pred q;\n\t.reg .u16 h;\n\tsetp.ne.s32 q, %2, 0;\n\tmov.u16 h, 0;\n\t@q ld.global.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}\n"
               : "=r"(v) : "l"(p), "r"((int)take) : "memory");
  return v;
}
__device__ __forceinline__ unsigned w4_ld_zero(const unsigned char* p, bool take) {
  unsigned v;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %2, 0;\n\tmov.u32 %0, 0;\n\t@q ld.global.u8 %0, [%1];\n\t}\n" : "=&r"(v) : "l"(p), "r"((int)take) : "memory");
  return v;
}

template <int MT, int WARPS, int U, int WORDS, bool ZEROS, typename TO>
__global__ void __launch_bounds__(WARPS * 32, 512 / (WARPS * 32))
gemm_w4_skinny_kernel(const bf16* __restrict__ x, long long ldx, const unsigned* __restrict__ w, long long ldw, const bf16* __restrict__ scales,
                      const unsigned char* __restrict__ zeros, int group, int groups, TO* __restrict__ out, long long ldo, int M, int N, int K,
                      int tiles, int trigger) {
  constexpr int CHUNK = 32 * WORDS;
  __shared__ float red[2][WARPS * MT * 32][4];
  if (trigger) pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int per_tile = ((K + CHUNK - 1) / CHUNK + WARPS - 1) / WARPS;          // chunks of a warp a tile, the last ones perhaps empty
  const int per_group = group / CHUNK;
  struct Slot { unsigned lo[WORDS], hi[WORDS], slo, shi, zlo, zhi; } slot[U];
  int tile = blockIdx.x, i = 0;                                                // what is asked for next: chunk i of this warp in the tile
  auto fetch = [&](Slot& s) {
    const int c = warp + i * WARPS, k = c * CHUNK + t * 8 * WORDS;
    const int n0 = tile * 16 + g < N ? tile * 16 + g : 0, n1 = tile * 16 + 8 + g < N ? tile * 16 + 8 + g : 0;   // rows beyond N stand for row 0
    const bool take = tile < tiles && k < K;
    w4_ld<WORDS>(w + (size_t)n0 * ldw + k / 8, take, s.lo);
    w4_ld<WORDS>(w + (size_t)n1 * ldw + k / 8, take, s.hi);
    const bool some = tile < tiles && c * CHUNK < K;
    const int at = some ? c / per_group : 0;
    const size_t a0 = (size_t)n0 * groups + at, a1 = (size_t)n1 * groups + at;
    s.slo = w4_ld_scale(scales + a0, some);
    s.shi = w4_ld_scale(scales + a1, some);
    if (ZEROS) { s.zlo = w4_ld_zero(zeros + a0, some); s.zhi = w4_ld_zero(zeros + a1, some); }
    if (++i == per_tile) { i = 0; tile += gridDim.x; }
  };
  for (int u = 0; u < U && u < per_tile; ++u) {                               // the first chunks' lines into L2: half a warp a lane, a row each
    const int n = tile * 16 + (lane & 15), k = (warp + u * WARPS) * CHUNK;
    if (lane < 16 && n < N && k < K) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(w + (size_t)n * ldw + k / 8) : "memory");
  }
  pdl_wait();
#pragma unroll
  for (int u = 0; u < U; ++u) fetch(slot[u]);
  float acc[MT][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
  int now = blockIdx.x, j = 0, par = 0;                                        // what is used next: chunk j of this warp in tile `now`
  while (now < tiles) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (now >= tiles) break;                                                 // alike for all warps of the block
      const int k = (warp + j * WARPS) * CHUNK + t * 8 * WORDS;
      Slot& s = slot[u];
      const __nv_bfloat162 blo = ZEROS ? w4_bias((int)s.zlo) : __float2bfloat162_rn(136.f), bhi = ZEROS ? w4_bias((int)s.zhi) : __float2bfloat162_rn(136.f);
      float part[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) part[mt][0] = part[mt][1] = part[mt][2] = part[mt][3] = 0.f;
#pragma unroll
      for (int q = 0; q < WORDS; ++q) {
        uint4 xv[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const bool in = mt * 8 + g < M;
          xv[mt] = w4_ld_x(x + (size_t)(in ? mt * 8 + g : 0) * ldx + k + 8 * q, in && k + 8 * q < K);
        }
        unsigned a[4], b[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) { a[p] = w4_pair(s.lo[q], p, blo); b[p] = w4_pair(s.hi[q], p, bhi); }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          w4_mma(part[mt], a[0], b[0], a[1], b[1], xv[mt].x, xv[mt].y);
          w4_mma(part[mt], a[2], b[2], a[3], b[3], xv[mt].z, xv[mt].w);
        }
      }
      const float slo = __uint_as_float(s.slo << 16), shi = __uint_as_float(s.shi << 16);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        acc[mt][0] += slo * part[mt][0]; acc[mt][1] += slo * part[mt][1];
        acc[mt][2] += shi * part[mt][2]; acc[mt][3] += shi * part[mt][3];
      }
      fetch(s);
      if (++j == per_tile) {                                                   // the tile is through: the warps' sums, added in warp order
        j = 0;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          *reinterpret_cast<float4*>(red[par][(warp * MT + mt) * 32 + lane]) = make_float4(acc[mt][0], acc[mt][1], acc[mt][2], acc[mt][3]);
          acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
        }
        __syncthreads();                       // one barrier a tile: a buffer is written again two tiles later, behind the next tile's barrier
        for (int idx = threadIdx.x; idx < MT * 128; idx += WARPS * 32) {
          const int mt = idx / 128, ln = (idx >> 2) & 31, e = idx & 3;
          float sum = 0.f;
#pragma unroll
          for (int v = 0; v < WARPS; ++v) sum += red[par][(v * MT + mt) * 32 + ln][e];
          const int n = now * 16 + (ln >> 2) + ((e >> 1) ? 8 : 0), m = mt * 8 + (ln & 3) * 2 + (e & 1);
          if (n < N && m < M) out[(size_t)m * ldo + n] = from_f32<TO>(sum);
        }
        par ^= 1;
        now += gridDim.x;
      }
    }
  }
}

template <int WORDS, bool ZEROS, typename TO>
static int w4_skinny(const W4Call& c) {
  const long long sms = si_sm_count(), tiles = (c.N + 15) / 16;
  int warps = 8;
  if (const char* e = getenv("W4_WARPS")) warps = atoi(e);
  const long long slots = 512 / (warps * 32) * sms;
  const dim3 grid((unsigned)(tiles > slots ? slots : tiles)), block(warps * 32);
  const int trig = si_pdl_trigger_mode(grid.x, slots);
  constexpr int U1 = WORDS == 4 ? 4 : 8, U2 = WORDS == 4 ? 3 : 6;
#define W4_SK(MT, WARPS, U) si_launch(gemm_w4_skinny_kernel<MT, WARPS, U, WORDS, ZEROS, TO>, grid, block, 0, c.stream, c.x, c.ldx, c.w, c.ldw, c.scales, \
                                      c.zeros, c.group, c.groups, (TO*)c.out, c.ldo, c.M, c.N, c.K, (int)tiles, trig)
  if (c.M > 8) { if (warps == 4) W4_SK(2, 4, U2); else W4_SK(2, 8, U2); }
  else if (warps == 4) W4_SK(1, 4, U1); else W4_SK(1, 8, U1);
#undef W4_SK
  return si_last_error();
}

template <typename TO>
static int w4_few(const W4Call& c) {
  if (c.group % 128 == 0) return c.zeros ? w4_skinny<4, true, TO>(c) : w4_skinny<4, false, TO>(c);
  if (c.group == 64) return c.zeros ? w4_skinny<2, true, TO>(c) : w4_skinny<2, false, TO>(c);
  return c.zeros ? w4_skinny<1, true, TO>(c) : w4_skinny<1, false, TO>(c);
}

// ---- more than 16 rows -------------------------------------------------------------------------------------------
// out transposed: a tile is HALVES x 128 rows of the weight matrix (the M of the instruction) by `bn` rows of x (its N, a multiple of 16), k steps
// of 128. Warp 0 fetches x (two boxes of 64 entries a step, 128-byte swizzle), warp 1 the words (rows of 64 bytes, 64-byte swizzle), both into one
// ring. Warps 8 to 15 widen: a thread owns one row of the weight matrix, takes its 64 bytes of a step out of shared memory (the swizzle spreads
// eight rows over all banks), makes the 128 entries bf16 in registers and writes them to its lane of tensor memory, from where the instruction reads
// its A: the widened weights cost neither bandwidth nor room in shared memory. Two groups of four warps take the steps in turn (HALVES 1) or a
// half of the rows each (HALVES 2, for few rows of x, where a step's instructions are short and its fixed cost counts). Warp 2 issues; warps
// 4 to 7 store. Tensor memory: with bn up to 192 two accumulators and two A buffers, beyond one and four (HALVES 2: up to 64 two, else one, and
// two A buffers a half). Blocks are persistent, one an SM; with few tiles the k range of a tile is cut over a cluster, whose blocks leave their
// sums in shared memory and add a part of the rows each up over all blocks, in their order.
#define W4_TC_SMEM (224 * 1024)
#define W4_TC_MAX_STAGES 8

__host__ __device__ inline int w4_tc_stage_bytes(int halves, int bn) { return halves * 128 * 64 + bn * 256; }
__host__ __device__ inline int w4_tc_stages(int halves, int bn) {
  const int n = W4_TC_SMEM / w4_tc_stage_bytes(halves, bn);
  return n < W4_TC_MAX_STAGES ? n : W4_TC_MAX_STAGES;
}
__device__ __forceinline__ float4 w4_ld_cluster(unsigned cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ void w4_drain(uint64_t* full, int stages, int issued) {       // as drain_copies in gemm_q8.cu
  for (int i = issued > stages ? issued - stages : 0; i < issued; ++i) mbar_wait(&full[i % stages], (unsigned)((i / stages) & 1));
}

template <int HALVES, bool ZEROS, typename TO>
__global__ void __launch_bounds__(512, 1)
gemm_w4_tc_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const bf16* __restrict__ scales,
                  const unsigned char* __restrict__ zeros, int group, int groups, TO* __restrict__ out, long long ldo, int M, int N, int K, int bn,
                  int m_tiles, int parts, int* status) {
  constexpr int BK = 128, ROWS = HALVES * 128, W_BYTES = ROWS * 64;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t full_bar[W4_TC_MAX_STAGES], empty_bar[W4_TC_MAX_STAGES], a_full[4], a_empty[4], acc_full[2], acc_empty[2];
  __shared__ unsigned tmem_slot;
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int X_BYTES = bn * 256, STAGES = w4_tc_stages(HALVES, bn);
  unsigned char* Ws = smem;
  unsigned char* Xs = smem + STAGES * W_BYTES;
  float* partial = reinterpret_cast<float*>(smem);         // [bn][ROWS] once the operands are used up (at most 128 KB)
  const int nk = (K + BK - 1) / BK, tiles = (N + ROWS - 1) / ROWS * m_tiles;
  const int part = (int)cluster_cta_rank(), first = blockIdx.x / parts, stride = gridDim.x / parts;
  const int k0 = (int)((long long)nk * part / parts), steps = (int)((long long)nk * (part + 1) / parts) - k0;
  // columns of tensor memory
  const int acc_w = HALVES == 2 ? (bn <= 64 ? 64 : 128) : (bn <= 192 ? 192 : 256);
  const int nbuf = HALVES == 2 ? (bn <= 64 ? 2 : 1) : (bn <= 192 ? 2 : 1);
  const int a_bufs = HALVES == 2 ? 2 : (bn <= 192 ? 2 : 4), a_col = HALVES == 2 ? 256 : (bn <= 192 ? 384 : 256);
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 2); mbar_init(&empty_bar[s], 1); }
#pragma unroll
    for (int b = 0; b < 4; ++b) { mbar_init(&a_full[b], 4 * HALVES); mbar_init(&a_empty[b], 1); }
#pragma unroll
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 4); }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 3) tmem_alloc(&tmem_slot, 512);
  tc05_fence_before_sync();
  __syncthreads();
  tc05_fence_after_sync();
  const unsigned tmem = tmem_slot;
  if (warp < 2) {
    if (lane == 0) {
      const bool is_w = warp == 1;
      const int bytes = is_w ? W_BYTES : X_BYTES;
      unsigned char* ring = is_w ? Ws : Xs;
      if (is_w && first < tiles)
        for (int i = 0; i < steps && i < STAGES; ++i)
          asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n"
                       ::"l"(&wmap), "r"((k0 + i) * (BK / 8)), "r"(first / m_tiles * ROWS) : "memory");
      pdl_wait();
      int s = 0, issued = 0;
      unsigned phase = 1;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        const int y = is_w ? tile / m_tiles * ROWS : tile % m_tiles * bn;
        for (int it = 0; it < steps; ++it, ++issued) {
          if (issued >= STAGES && !mbar_wait(&empty_bar[s], phase)) {
            set_status(status, SI_WAIT_LIMIT);
            w4_drain(full_bar, STAGES, issued);
            ok = false;
            break;
          }
          unsigned char* to = ring + s * bytes;
          mbar_expect_tx(&full_bar[s], (unsigned)bytes);   // both warps arrive, each with its own bytes
          if (is_w) {
            tma_load_2d(to, &wmap, &full_bar[s], (k0 + it) * (BK / 8), y);
          } else {
            tma_load_2d(to, &xmap, &full_bar[s], (k0 + it) * BK, y);
            tma_load_2d(to + bytes / 2, &xmap, &full_bar[s], (k0 + it) * BK + 64, y);
          }
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 2) {
    const unsigned idesc = umma_idesc_bf16(128, bn, false);
    const unsigned long long xd0 = umma_desc_sw128(Xs, 16, 1024);
    const unsigned x_step = (unsigned)X_BYTES / 16;
    int s = 0, b = 0, local = 0;
    unsigned phase = 0, a_phase = 0;
    unsigned long long xd = xd0;
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += stride, ++local) {
      const int d = nbuf == 2 ? local & 1 : 0;
      if (local >= nbuf) ok = mbar_wait_warp(&acc_empty[d], (unsigned)((local / nbuf - 1) & 1));
      if (!ok) break;
      tc05_fence_after_sync();
      const unsigned acc = tmem + (unsigned)(d * HALVES * acc_w);
      for (int it = 0; it < steps; ++it) {
        ok = mbar_wait_warp(&full_bar[s], phase) && mbar_wait_warp(&a_full[b], a_phase);
        if (!ok) break;
        tc05_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf) {
            const unsigned a = tmem + (unsigned)(a_col + (hf * 2 + b) * 64);          // HALVES 1: hf is 0
#pragma unroll
            for (int k = 0; k < 8; ++k)
              tc05_mma_bf16_tmem_a(acc + hf * acc_w, a + 8 * k, xd + (k >> 2) * (x_step / 2) + 2 * (k & 3), idesc, (it | k) != 0 ? 1u : 0u);
          }
          tc05_commit(&empty_bar[s]);
          tc05_commit(&a_empty[b]);
          if (it + 1 == steps) tc05_commit(&acc_full[d]);
        }
        __syncwarp();
        xd += x_step;
        if (++s == STAGES) { s = 0; xd = xd0; phase ^= 1u; }
        if (++b == a_bufs) { b = 0; a_phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
  } else if (warp >= 8) {
    const int g = (warp - 8) >> 2, row = (warp & 3) * 32 + lane, hf = HALVES == 2 ? g : 0;
    const unsigned char* wrow = Ws + (hf * 128 + row) * 64;
    const int swz = (row >> 1) & 3;
    const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
    const int every = HALVES == 2 ? 1 : 2;                 // this group's steps: every one, or every second one
    int s = 0, b = 0, st = 0;                              // of the step that comes next, over all tiles
    unsigned phase = 0, a_phase = 1;
    bool ok = true;
    pdl_wait();
    for (int tile = first; tile < tiles && ok; tile += stride) {
      const int n = tile / m_tiles * ROWS + hf * 128 + row;
      const bf16* srow = scales + (size_t)(n < N ? n : 0) * groups;
      const unsigned char* zrow = ZEROS ? zeros + (size_t)(n < N ? n : 0) * groups : nullptr;
      // scales of the four pieces of 32 entries of a step, asked for a step of this group ahead
      unsigned sc[4], zp[4];
      auto ask = [&](int it) {
        const int k = (k0 + it) * BK;
        if (group >= BK) {
          const int at = min(k / group, groups - 1);
          sc[0] = w4_ld_scale(srow + at, true);
          if (ZEROS) zp[0] = w4_ld_zero(zrow + at, true);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = min((k + 32 * j) / group, groups - 1);       // group is 32 or 64 here
            sc[j] = w4_ld_scale(srow + at, true);
            if (ZEROS) zp[j] = w4_ld_zero(zrow + at, true);
          }
        }
      };
      const int it0 = HALVES == 2 || (st & 1) == g ? 0 : 1;               // this group's first step of the tile
      if (it0 < steps) ask(it0);
      for (int it = 0; it < steps; ++it, ++st) {
        const bool mine = HALVES == 2 || (st & 1) == g;
        if (mine) {
          unsigned now[4], z[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) { now[j] = group >= BK ? sc[0] : sc[j]; z[j] = ZEROS ? (group >= BK ? zp[0] : zp[j]) : 8u; }
          if (it + every < steps) ask(it + every);
          ok = mbar_wait_warp(&full_bar[s], phase);
          if (!ok) break;
          uint4 wv[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) wv[j] = *reinterpret_cast<const uint4*>(wrow + s * W_BYTES + ((j ^ swz) << 4));
          if (st >= a_bufs) ok = mbar_wait_warp(&a_empty[b], a_phase);
          if (!ok) break;
          tc05_fence_after_sync();
          const unsigned a = tmem + lanes + (unsigned)(a_col + (hf * 2 + b) * 64);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            unsigned v[32];
#pragma unroll
            for (int j2 = 0; j2 < 2; ++j2) {
              const int j = 2 * h + j2;
              const __nv_bfloat162 bias = w4_bias((int)z[j]);
              const unsigned s2 = now[j] | (now[j] << 16);
              const unsigned words[4] = {wv[j].x, wv[j].y, wv[j].z, wv[j].w};
#pragma unroll
              for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                  const unsigned e = w4_pair(words[q], p, bias);
                  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&e), *reinterpret_cast<const __nv_bfloat162*>(&s2));
                  v[j2 * 16 + q * 4 + p] = *reinterpret_cast<const unsigned*>(&r);
                }
            }
            tmem_st_32x32_issue(a + h * 32, v);
          }
          tmem_st_wait();
          tc05_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&a_full[b]);
        }
        if (++s == STAGES) { s = 0; phase ^= 1u; }
        if (++b == a_bufs) { b = 0; a_phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
  } else if (warp >= 4) {
    pdl_wait();
    const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
    const bool vec2 = ldo % 2 == 0 && (uintptr_t)out % (2 * sizeof(TO)) == 0;
    int local = 0;
    for (int tile = first; tile < tiles; tile += stride, ++local) {
      const int d = nbuf == 2 ? local & 1 : 0;
      const int m_base = tile % m_tiles * bn, n_base = tile / m_tiles * ROWS + (warp & 3) * 32;
      if (!mbar_wait_warp(&acc_full[d], (unsigned)((local / nbuf) & 1))) {
        if (lane == 0) set_status(status, SI_WAIT_LIMIT);
        break;
      }
      tc05_fence_after_sync();
      const int rows = min(bn, M - m_base);
#pragma unroll 1
      for (int hf = 0; hf < HALVES; ++hf) {
        const unsigned src = tmem + lanes + (unsigned)((d * HALVES + hf) * acc_w);
        const int n = n_base + hf * 128 + lane;
#pragma unroll 1
        for (int m0 = 0; m0 < bn; m0 += 32) {
          float v[32];
          tmem_ld_32x32(src + m0, v);
          if (hf == HALVES - 1 && m0 + 32 >= bn) {         // in registers: the issuer may have the accumulator back
            tc05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[d]);
          }
          if (parts > 1) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (m0 + j < bn) partial[(m0 + j) * ROWS + hf * 128 + (warp & 3) * 32 + lane] = v[j];
          } else if (vec2 && n_base + hf * 128 + 32 <= N) {
            // neighbouring lanes swap: the even one stores columns n, n + 1 of row j, the odd one of row j + 1
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float give = lane & 1 ? v[j] : v[j + 1], got = __shfl_xor_sync(0xffffffffu, give, 1);
              const float a = lane & 1 ? got : v[j], c = lane & 1 ? v[j + 1] : got;
              const int m = m0 + j + (lane & 1);
              if (m < rows) {
                TO* dst = out + (size_t)(m_base + m) * ldo + (n & ~1);
                if constexpr (sizeof(TO) == 4) *reinterpret_cast<float2*>(dst) = make_float2(a, c);
                else *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(a, c);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (m0 + j < rows && n < N) out[(size_t)(m_base + m0 + j) * ldo + n] = from_f32<TO>(v[j]);
          }
        }
      }
    }
  }
  if (parts > 1) {                                         // one tile a cluster
    __syncwarp();
    cluster_sync_all();                                    // every block's sums lie in its shared memory
    const int m_base = first % m_tiles * bn, n0 = first / m_tiles * ROWS;
    const int lo = bn * part / parts, hi = min(M - m_base, bn * (part + 1) / parts);
    const bool vec = ldo % 4 == 0 && (uintptr_t)out % 16 == 0;
    for (int i = threadIdx.x; i < (hi - lo) * (ROWS / 4); i += 512) {
      const int m = lo + i / (ROWS / 4), c4 = i % (ROWS / 4) * 4, n = n0 + c4;
      const float* at = partial + m * ROWS + c4;
      float4 v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = c < parts ? w4_ld_cluster(cluster_map_u32(at, (unsigned)c)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 1; c < 8; ++c) { v[0].x += v[c].x; v[0].y += v[c].y; v[0].z += v[c].z; v[0].w += v[c].w; }
      TO* dst = out + (size_t)(m_base + m) * ldo + n;
      if (vec && n + 4 <= N) {
        if constexpr (sizeof(TO) == 4) {
          *reinterpret_cast<float4*>(dst) = v[0];
        } else {
          __nv_bfloat162 p[2] = {__floats2bfloat162_rn(v[0].x, v[0].y), __floats2bfloat162_rn(v[0].z, v[0].w)};
          *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(p);
        }
      } else {
        const float r[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) if (n + j < N) dst[j] = from_f32<TO>(r[j]);
      }
    }
    cluster_sync_all();                                    // no block goes while another one reads its sums
  }
  tc05_fence_before_sync();
  __syncthreads();
  if (warp == 3) tmem_dealloc(tmem, 512);
}

struct W4Shape { int halves, bn, m_tiles, parts; };

static void w4_tc_config(cudaLaunchConfig_t* cfg, unsigned blocks, int parts, cudaStream_t stream, cudaLaunchAttribute* attr) {
  cfg->gridDim = dim3(blocks);
  cfg->blockDim = dim3(512);
  cfg->dynamicSmemBytes = W4_TC_SMEM + 1024;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attr;
  cfg->numAttrs = si_pdl_enabled() ? 2 : 1;
}

// Clusters of `parts` blocks that the device runs at once, asked once per device and size (all forms of the kernel take an SM a block).
static int w4_clusters(int parts) {
  static int known[64][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (parts == 1) return si_sm_count();
  if (!known[dev][parts]) {
    auto k = gemm_w4_tc_kernel<1, true, bf16>;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = {};
    w4_tc_config(&cfg, (unsigned)parts, parts, 0, attr);
    int n = 0;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_TC_SMEM + 1024) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = 1; }
    known[dev][parts] = n;
  }
  return known[dev][parts];
}

static W4Shape w4_shape(int M, int N, int K) {
  const int nk = (K + 127) / 128;
  W4Shape best = {1, 128, 1, 1};
  double least = -1;
  for (int halves = 1; halves <= 2; ++halves) {
    if (halves == 2 && M > 128) break;
    const int n_tiles = (N + halves * 128 - 1) / (halves * 128);
    const int fewest = (M + 255) / 256;
    for (int mt = fewest; mt <= fewest + 2; ++mt) {
      const int bn = ((M + mt - 1) / mt + 15) / 16 * 16;
      if (mt > fewest && bn < 96) break;
      for (int parts = 1; parts <= 8 && parts <= nk; parts *= 2) {
        const long long tiles = (long long)n_tiles * mt, slots = w4_clusters(parts);
        if (parts > 1 && tiles > slots) break;
        const int steps = (nk + parts - 1) / parts;
        const double mma = (bn / 2 > 47 ? bn / 2 : 47) * 8.0 * halves, step = halves == 2 ? (mma + 420 > 900 ? mma + 420 : 900) : (mma + 100 > 600 ? mma + 100 : 600);
        const bool one = halves == 1 && bn > 192;
        const double cost = (double)((tiles + slots - 1) / slots) * (steps * step + (one ? 20.0 * bn : 500.0)) + 6000 + 16.0 * bn + (parts > 1 ? 2500 : 0);
        if (least < 0 || cost < least) { least = cost; best = W4Shape{halves, bn, mt, parts}; }
      }
    }
  }
  if (const char* e = getenv("W4_SHAPE")) sscanf(e, "%d,%d,%d,%d", &best.halves, &best.bn, &best.m_tiles, &best.parts);
  if (getenv("W4_SAY")) printf("shape %dx%dx%d: halves %d bn %d mt %d parts %d\n", M, N, K, best.halves, best.bn, best.m_tiles, best.parts);
  return best;
}

static int w4_encode(CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, long long rows, long long cols, long long ld, unsigned box_cols,
                     unsigned box_rows, CUtensorMapSwizzle swizzle) {
  SiEncodeTiledFn fn = si_encode_fn();
  if (!fn) return -3;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
  const cuuint32_t box[2] = {box_cols, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

template <int HALVES, bool ZEROS, typename TO>
static int w4_tc_launch(const W4Call& c, const W4Shape& sh) {
  auto k = gemm_w4_tc_kernel<HALVES, ZEROS, TO>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_TC_SMEM + 1024);
  if (e != cudaSuccess) return (int)e;
  CUtensorMap xm, wm;
  int rc = w4_encode(&xm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, c.x, c.M, c.K, c.ldx, 64, (unsigned)sh.bn, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = w4_encode(&wm, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, c.w, c.N, c.K / 8, c.ldw, 16, HALVES * 128, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc) return rc;
  const long long tiles = (long long)((c.N + HALVES * 128 - 1) / (HALVES * 128)) * sh.m_tiles, slots = si_sm_count();
  if (tiles > 0x0fffffffLL) return -2;
  const long long blocks = sh.parts > 1 ? tiles * sh.parts : tiles < slots ? tiles : slots;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  w4_tc_config(&cfg, (unsigned)blocks, sh.parts, c.stream, attr);
  cudaLaunchKernelEx(&cfg, k, xm, wm, c.scales, c.zeros, c.group, c.groups, (TO*)c.out, c.ldo, c.M, c.N, c.K, sh.bn, sh.m_tiles, sh.parts, c.status);
  return si_last_error();
}

template <typename TO>
static int w4_tc(const W4Call& c) {
  const W4Shape sh = w4_shape(c.M, c.N, c.K);
  if (sh.halves == 2) return c.zeros ? w4_tc_launch<2, true, TO>(c, sh) : w4_tc_launch<2, false, TO>(c, sh);
  return c.zeros ? w4_tc_launch<1, true, TO>(c, sh) : w4_tc_launch<1, false, TO>(c, sh);
}

// 1 when these kernels take operands so laid out (rows that start on 16-byte boundaries and end on one, the driver's tensor maps), else
// gemm_quant.cu does.
SI_EXPORT int si_gemm_w4_ok(const void* x, long long ldx, const void* w, long long ldw, int K) {
  return si_encode_fn() != nullptr && ((uintptr_t)x | (uintptr_t)w) % 16 == 0 && ldx % 8 == 0 && ldw % 4 == 0 && K % 32 == 0 && ldx >= K && ldw >= K / 8;
}

// x [M, K] bf16, rows `ldx` apart; w [N, K / 8] int32 words, rows `ldw` words apart; scales bf16 [N, ceil(K / group)], zeros uint8 like them or null;
// group 32, 64 or a multiple of 128; out [M, N], rows `ldo` apart, SI_BF16 or SI_F32. Returns 0, a CUDA error code, or -2 (size or layout refused).
SI_EXPORT int si_gemm_w4(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, int group, void* out,
                         long long ldo, int out_dtype, int M, int N, int K, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 8 || K > 0x3fffffff || !(group == 32 || group == 64 || (group > 0 && group % 128 == 0)) || !si_gemm_w4_ok(x, ldx, w, ldw, K)) return -2;
  W4Call c;
  c.x = (const bf16*)x; c.ldx = ldx; c.w = (const unsigned*)w; c.ldw = ldw; c.scales = (const bf16*)scales; c.zeros = (const unsigned char*)zeros;
  c.group = group; c.groups = (K - 1) / group + 1; c.out = out; c.ldo = ldo; c.M = M; c.N = N; c.K = K; c.status = status; c.stream = stream;
  if (M <= 16) return out_dtype == SI_BF16 ? w4_few<bf16>(c) : w4_few<float>(c);
  return out_dtype == SI_BF16 ? w4_tc<bf16>(c) : w4_tc<float>(c);
}
