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
  return -2;
}
