// Product of bf16 rows with 4-bit weights: out[m, n] = sum_k x[m, k] * s[n, k / group] * (q[n, k] - z[n, k / group]), sums fp32, bf16 or fp32
// output. q lies in int32 words of eight entries (quant_common.cuh); the weights are widened in registers on their way to the tensor cores and
// never written anywhere in between. Two kernels by the number of rows:
//   up to 8 rows, K a multiple of 256 up to 32,768    a stream of the weights through the fragments of mma.sync; q - z is exact in bf16, and with groups
//                    of 128 and more the scale is applied to the fp32 sum of a group, so that no weight is rounded
//   else             tcgen05 the other way round: 128 rows of the weight matrix are the M of the instruction and come to it through tensor memory,
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

// ---- up to 8 rows ------------------------------------------------------------------------------------------------
// mma.sync m16n8k16 with 16 rows of the weight matrix (a unit) as its "m" and the rows of x as its "n". A block a SM goes through its units; sixteen
// warps take a piece of 256 entries of the unit's rows each, always the same one of the block's at most 4,096, so that a warp's part of x stays in its
// registers. All that is not arithmetic is kept away from them: one TMA load brings a unit, [16 pieces][16 rows][128 bytes] (128-byte swizzle), into a
// ring of stages, four more warps bring the scales (and zero points), and four add the sixteen warps' sums of a unit up and store them.
// Lane (g, t) holds entries 32 t .. 32 t + 31 of a chunk of 128 of rows r(g) and r(g) + 8, r(g) = 4 (g mod 2) + g / 2 (neighbouring g then lie in different
// halves of the swizzle: no bank conflict), and the same entries of row g of x. A word's four pairs are the k columns of two instructions, alike
// for both operands. Groups of 128 and more: a chunk lies in one group, its sums are scaled by the row's number and added to the running ones, and
// no weight is rounded. SMALL (groups of 64 and 32): a lane's entries lie in one group, and a weight times its scale is rounded to bf16 (by 2^-8 of
// it at most), as with more rows.
//
// Eight rows of 28,672 x 4,096 take 16.8 us (3.5 TB/s), 17.5 with zero points, 18.3 and 20.1 with groups of 64 or 32. What bounds it is not told apart.
// Not memory (34 % of its rate) and not the tensor pipe (15 %); taking entries apart costs three shifts, four masks and four subtractions for eight weights,
// all but fp32 instructions issue every second clock (ALU 51 %), but without the subtractions it was no faster (below). A unit's full wait and exchange of
// sums, and 13 units for the busiest SM where 12.1 would be its share, are the rest. Other forms, us: words
// and x by loads of the lanes, the next words on their way to registers 27.9 and, with all arithmetic taken out, still 23 (a register that a load is to fill
// cannot be moved); words by a TMA load of every warp's own, scales by its lanes 28.3, 240 instructions a chunk, 130 of them not the product's; by one TMA
// load a unit and warps for the scales, x in shared memory, the sums added by the same warps behind a barrier 21.9, 203 instructions. Sums that start at
// -(128 + z) times those of x, without the subtractions: 16.6, but 3.6 for 3.4 at 2,048 x 2,048, and an infinity in x gives NaN. Scales asked for three
// units ahead: 16.7.
//
// More than 4,096 entries a row: a cluster shares the units, each block with its slice of k; the sums of all units wait in
// shared memory until the cluster meets, and each block adds up and stores every parts-th unit, in the order of the blocks.
#define W4_FEW_ROWS 8
#define W4_FEW_WARPS 16
#define W4_FEW_HELPERS 4                                    // warps that bring scales, and as many that add sums up
#define W4_FEW_THREADS ((W4_FEW_WARPS + 2 * W4_FEW_HELPERS) * 32)
#define W4_FEW_SLICE 4096
#define W4_FEW_STAGE (16 * 2048)
#define W4_FEW_SMEM (208 * 1024)                           // beside it the warps' sums, 16 KB
__device__ __forceinline__ void w4_mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Loads of what the kernels before may have written: not by the read-only path, whose loads may be moved across the wait for them.
__device__ __forceinline__ uint4 w4_ld_x(const bf16* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned w4_ld_scale(const bf16* p) {
  unsigned short v;
  asm volatile("ld.global.u16 %0, [%1];\n" : "=h"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned w4_ld_zero(const unsigned char* p) {
  unsigned v;
  asm volatile("ld.global.u8 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 w4_ld_8(const void* p) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned w4_ld_4(const void* p) {
  unsigned v;
  asm volatile("ld.global.u32 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float w4_ld_cluster1(unsigned cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}
// The first 1,024-byte boundary of dynamic shared memory. (Not by rounding the pointer itself, of which the compiler then no longer knows that it leads to
// shared memory.)
__device__ __forceinline__ unsigned char* w4_smem_base(unsigned char* smem) { return smem + ((1024u - (tma_smem_u32(smem) & 1023u)) & 1023u); }
// A wait that all lanes of a warp make, with one answer.
__device__ __forceinline__ bool w4_wait(uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

// Scales a row and stage as they lie in shared memory: one a chunk of 128, or (SMALL) one a piece of 32.
__host__ __device__ constexpr int w4_few_scales(bool small) { return small ? 128 : 32; }
__host__ __device__ constexpr int w4_few_stage_bytes(bool zeros, bool small) { return W4_FEW_STAGE + 16 * w4_few_scales(small) * (zeros ? 3 : 2); }
#define W4_FEW_STAGES 4

template <bool ZEROS, bool SMALL, typename TO>
__global__ void __launch_bounds__(W4_FEW_THREADS, 1)
gemm_w4_few_kernel(const __grid_constant__ CUtensorMap wmap, const bf16* __restrict__ x, long long ldx, const bf16* __restrict__ scales,
                   const unsigned char* __restrict__ zeros, int group, int groups, TO* __restrict__ out, long long ldo, int M, int N, int K, int slice,
                   int parts, int units, int* status, int trigger) {
  constexpr int STAGES = W4_FEW_STAGES, SC = w4_few_scales(SMALL);
  extern __shared__ unsigned char smem_dyn[];
  __shared__ float red[2][W4_FEW_WARPS][128];
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], red_full[2], red_empty[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* ring = w4_smem_base(smem_dyn);
  unsigned short* sring = reinterpret_cast<unsigned short*>(ring + STAGES * W4_FEW_STAGE);     // [stage][16 rows][SC]
  unsigned char* zring = reinterpret_cast<unsigned char*>(sring + STAGES * 16 * SC);           // likewise
  float* sums = reinterpret_cast<float*>(ring + STAGES * w4_few_stage_bytes(ZEROS, SMALL));     // [unit][128], only where a cluster meets
  const int part = (int)cluster_cta_rank(), first = blockIdx.x / parts, stride = gridDim.x / parts;
  const int k_begin = part * slice, boxes = (min(K, k_begin + slice) - k_begin) / 256;         // K and slices are multiples of 256, none empty
  const int mine = (units - first + stride - 1) / stride;                                      // units of this block (first < units)
  if (trigger) pdl_trigger();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1 + W4_FEW_HELPERS); mbar_init(&empty_bar[s], W4_FEW_WARPS); }
#pragma unroll
    for (int b = 0; b < 2; ++b) { mbar_init(&red_full[b], W4_FEW_WARPS); mbar_init(&red_empty[b], W4_FEW_HELPERS); }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  bool ok = true;
  auto place = [&](int unit, int e, int* m, int* n) {         // row and column of sum e of a unit
    const int ln = e >> 2, g = ln >> 2;
    *m = (ln & 3) * 2 + (e & 1);
    *n = (first + unit * stride) * 16 + (g & 1) * 4 + (g >> 1) + ((e >> 1) & 1) * 8;
  };
  if (warp >= W4_FEW_WARPS + W4_FEW_HELPERS) {                // adds the warps' sums up, in their order, a thread one
    const int e = threadIdx.x - (W4_FEW_WARPS + W4_FEW_HELPERS) * 32;
    pdl_wait();                                               // `out` may still be read by the kernel before
    for (int unit = 0; unit < mine; ++unit) {
      const int par = unit & 1;
      ok = w4_wait(&red_full[par], (unsigned)((unit >> 1) & 1));
      if (!ok) break;
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < W4_FEW_WARPS; ++v) sum += red[par][v][e];
      if (parts > 1) {
        sums[unit * 128 + e] = sum;
      } else {
        int m, n;
        place(unit, e, &m, &n);
        if (n < N && m < M) out[(size_t)m * ldo + n] = from_f32<TO>(sum);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&red_empty[par]);
    }
  } else if (warp >= W4_FEW_WARPS) {
    const int b = warp - W4_FEW_WARPS;                        // brings the scales of rows 4 b .. 4 b + 3; the first of them the words as well
    const int pieces = slice / 256;
    if (b == 0 && lane == 0)
      asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];\n" ::"l"(&wmap), "r"(0), "r"(first * 16), "r"(k_begin / 256) : "memory");
    pdl_wait();
    int s = 0, issued = 0;
    unsigned phase = 1;
    for (int unit = 0; unit < mine; ++unit, ++issued) {
      const int u0 = (first + unit * stride) * 16;               // rows beyond N take row 0's scales: their words are zeros, nothing is stored
      // a row's scales of a stage, asked for before the stage is free. SMALL: eight pieces of 32 (a row's are whole vectors: K is a multiple of 256),
      // one scale each or one for two; else a chunk at a time, eight lanes a row
      uint4 sw[2];
      uint2 zw[2];
      unsigned sv[4], zv[4];
      if constexpr (SMALL) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = u0 + 4 * b + 2 * i + lane / 16, piece = k_begin / 32 + lane % 16 * 8;
          const size_t r = (size_t)(n < N ? n : 0) * groups;
          sw[i] = make_uint4(0, 0, 0, 0);
          zw[i] = make_uint2(0, 0);
          if (piece * 32 < K) {
            if (group == 32) {
              sw[i] = w4_ld_x(scales + r + piece);
              if (ZEROS) zw[i] = w4_ld_8(zeros + r + piece);
            } else {
              const uint2 h = w4_ld_8(scales + r + piece / 2);
              sw[i].x = h.x; sw[i].y = h.y;
              if (ZEROS) zw[i].x = w4_ld_4(zeros + r + piece / 2);
            }
          }
        }
      } else {
        const int n = u0 + 4 * b + lane / 8;
        const size_t r = (size_t)(n < N ? n : 0) * groups;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = min((k_begin + (lane % 8 + 8 * i) * 128) / group, groups - 1);
          sv[i] = w4_ld_scale(scales + r + at);
          if (ZEROS) zv[i] = w4_ld_zero(zeros + r + at);
        }
      }
      if (issued >= STAGES) ok = w4_wait(&empty_bar[s], phase);
      if (!ok) break;
      if (b == 0 && lane == 0) {
        mbar_expect_tx(&full_bar[s], (unsigned)pieces * 2048u);
        tma_load_3d(ring + s * W4_FEW_STAGE, &wmap, &full_bar[s], 0, u0, k_begin / 256);
      }
      if constexpr (SMALL) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = (s * 16 + 4 * b + 2 * i + lane / 16) * SC + lane % 16 * 8;
          if (group == 64) {                                     // one for two pieces; not sooner, the loads are still under way above
            const uint2 h = make_uint2(sw[i].x, sw[i].y);
            const unsigned q = zw[i].x;
            sw[i] = make_uint4(__byte_perm(h.x, 0, 0x1010), __byte_perm(h.x, 0, 0x3232), __byte_perm(h.y, 0, 0x1010), __byte_perm(h.y, 0, 0x3232));
            zw[i] = make_uint2(__byte_perm(q, 0, 0x1100), __byte_perm(q, 0, 0x3322));
          }
          *reinterpret_cast<uint4*>(sring + at) = sw[i];
          if (ZEROS) *reinterpret_cast<uint2*>(zring + at) = zw[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = (s * 16 + 4 * b + lane / 8) * SC + lane % 8 + 8 * i;
          sring[at] = (unsigned short)sv[i];
          if (ZEROS) zring[at] = (unsigned char)zv[i];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_bar[s]);
      if (++s == STAGES) { s = 0; phase ^= 1u; }
    }
    if (!ok && b == 0 && lane == 0)                             // the copies still under way, with a limit again
      for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i) mbar_wait(&full_bar[i % STAGES], (unsigned)((i / STAGES) & 1));
  } else {
    const int g = lane >> 2, t = lane & 3, row = (g & 1) * 4 + (g >> 1);
    const bool busy = warp < boxes;
    pdl_wait();
    uint4 xr[8];                                                // this warp's piece of x; a lane of a row that is not there takes row 0's: nothing of it is stored
    {
      const bf16* from = x + (size_t)(g < M ? g : 0) * ldx + k_begin + (busy ? warp : 0) * 256 + t * 32;
#pragma unroll
      for (int i = 0; i < 8; ++i) xr[i] = w4_ld_x(from + (i >> 2) * 128 + (i & 3) * 8);
    }
    const unsigned char* wl = ring + warp * 2048 + row * 128;
    const int off[2] = {(t ^ row) << 4, ((4 + t) ^ row) << 4};
    const int se = row * SC + (SMALL ? warp * 8 + t : warp * 2);        // this lane's scales of a stage: chunk h's 4 h (SMALL) or h further
    int s = 0;
    unsigned phase = 0;
#pragma unroll 1
    for (int unit = 0; unit < mine; ++unit) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      ok = w4_wait(&full_bar[s], phase);
      if (!ok) break;
      if (busy) {                                               // alike for the warp
        const unsigned char* box = wl + s * W4_FEW_STAGE;
        const unsigned short* sp = sring + s * 16 * SC + se;
        const unsigned char* zp = zring + s * 16 * SC + se;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int sh = SMALL ? 4 * h : h;
          const uint4 lo = *reinterpret_cast<const uint4*>(box + off[h]), hi = *reinterpret_cast<const uint4*>(box + 1024 + off[h]);
          const unsigned slo = sp[sh], shi = sp[8 * SC + sh];
          const __nv_bfloat162 blo = ZEROS ? w4_bias((int)zp[sh]) : __float2bfloat162_rn(136.f);
          const __nv_bfloat162 bhi = ZEROS ? w4_bias((int)zp[8 * SC + sh]) : __float2bfloat162_rn(136.f);
          const unsigned lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
          const unsigned s0w = slo | (slo << 16), s1w = shi | (shi << 16);
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 xv = xr[h * 4 + q];
            unsigned a[4], c[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              a[p] = w4_pair(lw[q], p, blo);
              c[p] = w4_pair(hw[q], p, bhi);
              if (SMALL) {
                const __nv_bfloat162 ra = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a[p]), *reinterpret_cast<const __nv_bfloat162*>(&s0w));
                const __nv_bfloat162 rc = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&c[p]), *reinterpret_cast<const __nv_bfloat162*>(&s1w));
                a[p] = *reinterpret_cast<const unsigned*>(&ra);
                c[p] = *reinterpret_cast<const unsigned*>(&rc);
              }
            }
            float (&to)[4] = SMALL ? acc : sum;
            w4_mma(to, a[0], c[0], a[1], c[1], xv.x, xv.y);
            w4_mma(to, a[2], c[2], a[3], c[3], xv.z, xv.w);
          }
          if (!SMALL) {
            const float s0 = __uint_as_float(slo << 16), s1 = __uint_as_float(shi << 16);
            acc[0] += s0 * sum[0]; acc[1] += s0 * sum[1];
            acc[2] += s1 * sum[2]; acc[3] += s1 * sum[3];
          }
        }
      }
      const int par = unit & 1;
      if (unit >= 2) {
        ok = w4_wait(&red_empty[par], (unsigned)(((unit >> 1) - 1) & 1));
        if (!ok) break;
      }
      *reinterpret_cast<float4*>(&red[par][warp][lane * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&red_full[par]);
        mbar_arrive(&empty_bar[s]);                             // a stage and a slot go back when what was read there has been used
      }
      if (++s == STAGES) { s = 0; phase ^= 1u; }
    }
  }
  if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
  if (parts > 1) {
    cluster_sync_all();                                         // every block's sums of its slice lie in its shared memory
    for (int i = threadIdx.x; i < mine * 128; i += W4_FEW_THREADS) {
      const int unit = i >> 7, e = i & 127;
      if (unit % parts != part) continue;
      float v[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) v[p] = p < parts ? w4_ld_cluster1(cluster_map_u32(sums + i, (unsigned)p)) : 0.f;
#pragma unroll
      for (int p = 1; p < 8; ++p) v[0] += v[p];
      int m, n;
      place(unit, e, &m, &n);
      if (n < N && m < M && ok) out[(size_t)m * ldo + n] = from_f32<TO>(v[0]);
    }
    cluster_sync_all();                                         // no block goes while another one reads its sums
  }
}

// How k is cut: blocks of a cluster, a block's slice, clusters, dynamic shared memory. False where it does not fit.
static int w4_clusters(int size);
struct W4Few { int parts, slice, clusters; size_t smem; };
static bool w4_few_shape(int M, int N, int K, bool zeros, bool small, W4Few* f) {
  if (M > W4_FEW_ROWS || K % 256) return false;
  const int units = (N + 15) / 16, boxes = K / 256;
  for (int parts = 1; parts <= 8; parts *= 2) {
    const int per = (boxes + parts - 1) / parts;
    if ((long long)per * (parts - 1) >= boxes) return false;                                    // a block without a piece
    if (per * 256 > W4_FEW_SLICE) continue;
    const int slots = w4_clusters(parts);
    f->parts = parts;
    f->slice = per * 256;
    f->clusters = units < slots ? units : slots;
    f->smem = (size_t)W4_FEW_STAGES * w4_few_stage_bytes(zeros, small) + 1024 + (parts > 1 ? (size_t)((units + f->clusters - 1) / f->clusters) * 512 : 0);
    return f->smem <= W4_FEW_SMEM;
  }
  return false;
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
// The words [rows, pieces of 128 bytes] as (word of a piece, row, piece), boxes of [box_pieces, 16 rows, 128 bytes].
static int w4_encode_pieces(CUtensorMap* map, const void* base, long long rows, int pieces, long long ld, int box_pieces) {
  SiEncodeTiledFn fn = si_encode_fn();
  if (!fn) return -3;
  const cuuint64_t dims[3] = {32, (cuuint64_t)rows, (cuuint64_t)pieces};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * 4), 128};
  const cuuint32_t box[3] = {32, 16, (cuuint32_t)box_pieces};
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

template <bool ZEROS, bool SMALL, typename TO>
static int w4_few_launch(const W4Call& c, const W4Few& f) {
  auto k = gemm_w4_few_kernel<ZEROS, SMALL, TO>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_FEW_SMEM);
  if (e != cudaSuccess) return (int)e;
  CUtensorMap wm;
  const int rc = w4_encode_pieces(&wm, c.w, c.N, c.K / 256, c.ldw, f.slice / 256);
  if (rc) return rc;
  const int blocks = f.clusters * f.parts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(W4_FEW_THREADS);
  cfg.dynamicSmemBytes = f.smem;
  cfg.stream = c.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)f.parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = si_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, k, wm, c.x, c.ldx, c.scales, c.zeros, c.group, c.groups, (TO*)c.out, c.ldo, c.M, c.N, c.K, f.slice, f.parts,
                     (c.N + 15) / 16, c.status, si_pdl_trigger_mode(blocks, si_sm_count()));
  return si_last_error();
}

template <typename TO>
static int w4_few(const W4Call& c, const W4Few& f) {
  if (c.group < 128) return c.zeros ? w4_few_launch<true, true, TO>(c, f) : w4_few_launch<false, true, TO>(c, f);
  return c.zeros ? w4_few_launch<true, false, TO>(c, f) : w4_few_launch<false, false, TO>(c, f);
}

// ---- more than 8 rows --------------------------------------------------------------------------------------------
// out transposed: a tile is 128 rows of the weight matrix a CTA (the M of the instruction) by `bn` rows of x (its N, a multiple of 16), k steps of 256.
// Two slots go round (three up to 64 rows of x); to a slot belong the step's part of x and 128 columns of tensor memory for the widened weights. Warp 0
// fetches x (boxes of 64 entries, 128-byte swizzle), warp 1 the words, half a step at a time (rows of 64 bytes, 64-byte swizzle), into eight stages of
// their own: given back with the slots, a load's way from memory stood between any two uses of one. Warps 8 to 23 widen, four to half a step, so that two
// steps are in the making at once (all but fp32 arithmetic issues every second clock, and one warp a scheduler left more than half of those empty): a
// thread owns one row of the weight matrix, takes its 64 bytes out of shared memory (the swizzle spreads eight rows over all banks), makes the 128 entries
// bf16 in registers and writes them to its lane of tensor memory, where the instruction reads its A: the widened weights cost neither bandwidth nor room in
// shared memory. Warp 2 issues, sixteen instructions a step; warps 4 to 7 store. Up to 128 rows of x there are two accumulators, beyond one of 256 columns.
//
// PAIR: two CTAs (a cluster) on a tile of 256 rows of the weight matrix, each with its 128 in its own tensor memory and half of the tile's rows of x; the
// leader's instructions (cta_group::2) read both. With many rows x is what bounds a CTA alone: it takes in bn * 256 bytes of it for every 8 KB of
// words, and an SM was seen to take in 50 to 80 GB/s (937 x 4,096 x 14,336: 81 us, 105 alone).
//
// A wait costs the issuing warp 100 to 350 clocks even where there is nothing to wait for, and a commit not less than that, so there is one of each
// a step: `ready` of a slot counts the bytes of x and the warps that widened (the leader's counts both CTAs'), and the one commit on `empty` gives back
// all that belongs to the slot.
//
// Blocks are persistent, one an SM. Without PAIR the k range of a tile may be cut over a cluster, whose blocks leave their sums in shared memory and
// add a part of the rows each up over all blocks, in their order.
#define W4_MAX_SLOTS 3
#define W4_THREADS (24 * 32)
#define W4_WORDS 8                                          // stages of words
#define W4_TC_SMEM (W4_WORDS * 128 * 64 + 2 * 128 * 512)    // two slots with 128 rows of x a CTA (three with 64 take less)

__device__ __forceinline__ float4 w4_ld_cluster(unsigned cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ void w4_mma_pair_tmem_a(unsigned d, unsigned a, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// An arrival at the leader's barrier. What it orders lies in tensor memory, which the tcgen05 fences on both sides see to, so it is a relaxed one: a
// release to the cluster waits for everything the warp has under way (the scales asked for ahead among it) and took 1,000 to 1,700 clocks a step, and
// arrivals at home passed on by a warp of their own cost a tenth to two fifths of the whole (300 x 4,096 x 4,096: 17.7 us as it is, 23.6).
__device__ __forceinline__ void w4_arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_map_u32(bar, 0)) : "memory");
}
// After a wait that ran out: the copies still under way are waited for, with a limit again, before the block's shared memory goes.
__device__ __forceinline__ void w4_drain(uint64_t* full, int stages, int issued) {
  for (int i = issued > stages ? issued - stages : 0; i < issued; ++i) mbar_wait(&full[i % stages], (unsigned)((i / stages) & 1));
}

// The scales and zero points of one row of the weight matrix along its steps of 128 entries: those of a step are asked for ahead, when the
// caller's step before it is done with. Groups of 128 and more: one of each a step, the group counted along; SMALL (64 and 32): one a piece of 32 entries.
template <bool ZEROS, bool SMALL> struct W4Scales {
  static constexpr int N = SMALL ? 4 : 1;
  const bf16* s; const unsigned char* z;
  int last, span, at, rem;              // last group; SMALL: groups a step, else steps a group; group of the next step, and its place in it
  unsigned sv[N], zv[N];
  __device__ __forceinline__ void start(const bf16* scales, const unsigned char* zeros, long long row, int group, int groups, int step) {
    last = groups - 1;
    s = scales + row * groups;
    z = ZEROS ? zeros + row * groups : nullptr;
    span = SMALL ? 128 / group : group / 128;
    at = SMALL ? step * span : step / span;
    rem = SMALL ? 0 : step % span;
  }
  // `by`: steps until the caller's next one
  __device__ __forceinline__ void ask(int by) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = min(SMALL ? at + (span == 4 ? j : j >> 1) : at, last);
      sv[j] = w4_ld_scale(s + i);
      if (ZEROS) zv[j] = w4_ld_zero(z + i);
    }
    if (SMALL) {
      at += by * span;
    } else {
      rem += by;
      while (rem >= span) { rem -= span; ++at; }
    }
  }
};

// A thread's row of a step, 128 entries, out of shared memory (64 bytes in the 64-byte swizzle: `swz` is the row's) ...
__device__ __forceinline__ void w4_take_row(const unsigned char* row, int swz, uint4 (&wv)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) wv[j] = *reinterpret_cast<const uint4*>(row + ((j ^ swz) << 4));
}
// ... as bf16 into 64 columns of its lane of tensor memory, a piece of 32 entries (16 columns) at a time. TAIL: the row ends `left` entries from here. What
// the step holds beyond stands for nothing, but its words are zeros, which the last group's zero point and scale may make infinite, and x's zeros with that
// NaN; so their scale is zero. (A form of its own: the choice of a scale a piece would be a thirtieth of the instructions of every step.)
template <bool ZEROS, bool SMALL, bool TAIL>
__device__ __forceinline__ void w4_widen_row(const uint4 (&wv)[4], const unsigned* scale, const unsigned* zero, unsigned a, int left) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = SMALL ? j : 0;
    const __nv_bfloat162 bias = ZEROS ? w4_bias((int)zero[i]) : __float2bfloat162_rn(136.f);
    const unsigned s2 = TAIL && 32 * j >= left ? 0u : scale[i] | (scale[i] << 16);
    const unsigned words[4] = {wv[j].x, wv[j].y, wv[j].z, wv[j].w};
    unsigned v[16];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const unsigned e = w4_pair(words[q], p, bias);
        const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&e), *reinterpret_cast<const __nv_bfloat162*>(&s2));
        v[q * 4 + p] = *reinterpret_cast<const unsigned*>(&r);
      }
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 ::"r"(a + j * 16), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                   "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
  }
  tmem_st_wait();
}

// 32 rows of x (from m0 on, `rows` of the tile in all) of this thread's column n of the output; `whole`: the warp's 32 columns lie inside. Neighbouring
// lanes swap, so that the even one stores columns n and n + 1 of one row and the odd one of the next.
template <typename TO>
__device__ __forceinline__ void w4_store(TO* __restrict__ out, long long ldo, const float (&v)[32], long long m_base, int m0, int rows, int n, int N, int lane,
                                         bool whole) {
  if (whole) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const float give = lane & 1 ? v[j] : v[j + 1], got = __shfl_xor_sync(0xffffffffu, give, 1);
      const float a = lane & 1 ? got : v[j], c = lane & 1 ? v[j + 1] : got;
      const int m = m0 + j + (lane & 1);
      if (m < rows) {
        TO* dst = out + (m_base + m) * ldo + (n & ~1);
        if constexpr (sizeof(TO) == 4) *reinterpret_cast<float2*>(dst) = make_float2(a, c);
        else *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(a, c);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (m0 + j < rows && n < N) out[(m_base + m0 + j) * ldo + n] = from_f32<TO>(v[j]);
  }
}

template <bool PAIR, bool ZEROS, bool SMALL, typename TO>
__global__ void __launch_bounds__(W4_THREADS, 1)
gemm_w4_tc_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const bf16* __restrict__ scales,
                  const unsigned char* __restrict__ zeros, int group, int groups, TO* __restrict__ out, long long ldo, int M, int N, int K, int bn,
                  int m_tiles, int parts, int* status, int trigger) {
  constexpr int BK = 256, W_BYTES = 128 * 64, CTAS = PAIR ? 2 : 1, ROWS = 128 * CTAS;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t w_full[W4_WORDS], w_empty[W4_WORDS], ready[W4_MAX_SLOTS], empty_bar[W4_MAX_SLOTS], acc_full[2], acc_empty[2];
  __shared__ unsigned tmem_slot;
  unsigned char* Ws = w4_smem_base(smem_dyn);
  unsigned char* Xs = Ws + W4_WORDS * W_BYTES;
  float* partial = reinterpret_cast<float*>(Ws);           // [bn][128] once the operands are used up (at most 128 KB)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_cta_rank() : 0, part = PAIR ? 0 : (int)cluster_cta_rank(), sharers = PAIR ? 2 : parts;
  const int X_BYTES = bn / CTAS * 512, slots = bn <= 64 ? 3 : 2;
  const int nk = (K + BK - 1) / BK, tiles = (N + ROWS - 1) / ROWS * m_tiles;
  const int k0 = (int)((long long)nk * part / parts), steps = (int)((long long)nk * (part + 1) / parts) - k0;
  const int first = blockIdx.x / sharers, stride = gridDim.x / sharers;
  const int nbuf = bn <= 128 ? 2 : 1, acc_w = bn <= 64 ? 64 : 128, a_col = bn <= 64 ? 128 : 256;      // columns of tensor memory: accumulators, then A
  if (trigger) pdl_trigger();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < W4_MAX_SLOTS; ++s) { mbar_init(&ready[s], 1 + 8 * CTAS); mbar_init(&empty_bar[s], 1); }
#pragma unroll
    for (int s = 0; s < W4_WORDS; ++s) { mbar_init(&w_full[s], 1); mbar_init(&w_empty[s], 4); }
#pragma unroll
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 4 * CTAS); }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 3) { if (PAIR) tmem_alloc_pair(&tmem_slot, 512); else tmem_alloc(&tmem_slot, 512); }
  tc05_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();       // both CTAs' barriers and tensor memory are ready
  tc05_fence_after_sync();
  const unsigned tmem = tmem_slot;
  if (warp < 2) {
    if (lane == 0) {
      const bool is_w = warp == 1;
      if (is_w && first < tiles)
        for (int i = 0; i < 2 * steps && i < W4_WORDS; ++i)
          asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n"
                       ::"l"(&wmap), "r"(k0 * (BK / 8) + i * 16), "r"(first / m_tiles * ROWS + rank * 128) : "memory");
      pdl_wait();
      // the words come half a step at a time, x a whole one
      const int stages = is_w ? W4_WORDS : slots, count = is_w ? 2 * steps : steps;
      uint64_t* free_bar = is_w ? w_empty : empty_bar;
      int s = 0, issued = 0;
      unsigned phase = 1;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        const int y = is_w ? tile / m_tiles * ROWS + rank * 128 : tile % m_tiles * bn + rank * (bn / 2);
        for (int it = 0; it < count; ++it, ++issued) {
          if (issued >= stages && !mbar_wait(&free_bar[s], phase)) {
            set_status(status, SI_WAIT_LIMIT);
            if (is_w) w4_drain(w_full, W4_WORDS, issued);
            else if (rank == 0) w4_drain(ready, slots, issued);
            ok = false;
            break;
          }
          if (is_w) {
            mbar_expect_tx(&w_full[s], W_BYTES);
            tma_load_2d(Ws + s * W_BYTES, &wmap, &w_full[s], k0 * (BK / 8) + it * 16, y);
          } else {
            unsigned char* to = Xs + s * X_BYTES;
            if (rank == 0) mbar_expect_tx(&ready[s], (unsigned)(CTAS * X_BYTES));
            const unsigned bar = cluster_map_u32(&ready[s], 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (PAIR) tma_load_2d_pair(to + j * (X_BYTES / 4), &xmap, bar, it * BK + 64 * j, y);
              else tma_load_2d(to + j * (X_BYTES / 4), &xmap, &ready[s], (k0 + it) * BK + 64 * j, y);
            }
          }
          if (++s == stages) { s = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 2) {
    if (rank == 0) {
      const unsigned idesc = umma_idesc_bf16(ROWS, bn, false);
      const unsigned long long xd0 = umma_desc_sw128(Xs, 16, 1024);
      const unsigned x_step = (unsigned)X_BYTES / 16;
      int s = 0, local = 0;
      unsigned phase = 0;
      unsigned long long xd = xd0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride, ++local) {
        const int d = nbuf == 2 ? local & 1 : 0;
        if (local >= nbuf) ok = w4_wait(&acc_empty[d], (unsigned)((local / nbuf - 1) & 1));
        if (!ok) break;
        tc05_fence_after_sync();
        const unsigned acc = tmem + (unsigned)(d * acc_w);
        for (int it = 0; it < steps; ++it) {
          ok = w4_wait(&ready[s], phase);
          if (!ok) break;
          tc05_fence_after_sync();
          if (elect_one()) {
            const unsigned a = tmem + (unsigned)(a_col + s * 128);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const unsigned long long b = xd + (k >> 2) * (x_step / 4) + 2 * (k & 3);
              if (PAIR) w4_mma_pair_tmem_a(acc, a + 8 * k, b, idesc, (it | k) != 0 ? 1u : 0u);
              else tc05_mma_bf16_tmem_a(acc, a + 8 * k, b, idesc, (it | k) != 0 ? 1u : 0u);
            }
            if (PAIR) tc05_commit_pair(&empty_bar[s], 3); else tc05_commit(&empty_bar[s]);
            if (it + 1 == steps) { if (PAIR) tc05_commit_pair(&acc_full[d], 3); else tc05_commit(&acc_full[d]); }
          }
          __syncwarp();
          xd += x_step;
          if (++s == slots) { s = 0; xd = xd0; phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) set_status(status, SI_WAIT_LIMIT);
    }
  } else if (warp >= 8) {
    // four groups of four warps take the half steps in turn; half h of a step goes to columns 64 h of the slot
    const int g = (warp - 8) >> 2, row = (warp & 3) * 32 + lane;
    const unsigned char* wrow = Ws + row * 64;
    const int swz = (row >> 1) & 3;
    const unsigned mine = tmem + ((unsigned)((warp & 3) * 32) << 16) + (unsigned)(a_col + (g & 1) * 64);
    int at = g;                                            // this group's next half step, counted from the tile's first
    int stage = g, turns = 0;                              // its words' stage (two in turn), and how many it has made
    int slot = g >> 1, uses = 0;                           // its slot, and how many times that was used before
    bool ok = true;
    pdl_wait();
    for (int tile = first; tile < tiles && ok; tile += stride, at -= 2 * steps) {
      const int n = tile / m_tiles * ROWS + rank * 128 + row;
      W4Scales<ZEROS, SMALL> sc;
      sc.start(scales, zeros, n < N ? n : 0, group, groups, 2 * k0 + at);
      if (at < 2 * steps) sc.ask(4);
      for (; at < 2 * steps; at += 4, ++turns, stage ^= 4) {
        unsigned now[W4Scales<ZEROS, SMALL>::N], z[W4Scales<ZEROS, SMALL>::N];
#pragma unroll
        for (int j = 0; j < W4Scales<ZEROS, SMALL>::N; ++j) { now[j] = sc.sv[j]; if (ZEROS) z[j] = sc.zv[j]; }
        if (at + 4 < 2 * steps) sc.ask(4);
        ok = w4_wait(&w_full[stage], (unsigned)((turns >> 1) & 1));
        if (!ok) break;
        uint4 wv[4];
        w4_take_row(wrow + stage * W_BYTES, swz, wv);
        if (uses > 0) ok = w4_wait(&empty_bar[slot], (unsigned)((uses - 1) & 1));
        if (!ok) break;
        tc05_fence_after_sync();
        const int left = K - (2 * k0 + at) * 128;            // a multiple of 32, as K is
        if (left >= 128) w4_widen_row<ZEROS, SMALL, false>(wv, now, z, mine + (unsigned)(slot * 128), left);
        else w4_widen_row<ZEROS, SMALL, true>(wv, now, z, mine + (unsigned)(slot * 128), left);
        tc05_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) w4_arrive_leader(&ready[slot]); else mbar_arrive(&ready[slot]);
          // Not before the words are used: given back as soon as they were in registers by the code's order, reads were seen to end up behind the wait
          // for the slot, after the stage's next words had come. Here their values have gone through the stores to tensor memory, and those are waited for.
          mbar_arrive(&w_empty[stage]);
        }
        slot += 2;
        if (slot >= slots) { slot -= slots; ++uses; }
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
      const int m_base = tile % m_tiles * bn, n_base = tile / m_tiles * ROWS + rank * 128 + (warp & 3) * 32;
      if (!mbar_wait_warp(&acc_full[d], (unsigned)((local / nbuf) & 1))) {
        if (lane == 0) set_status(status, SI_WAIT_LIMIT);
        break;
      }
      tc05_fence_after_sync();
      const int rows = min(bn, M - m_base);
#pragma unroll 1
      for (int m0 = 0; m0 < bn; m0 += 32) {
        float v[32];
        __syncwarp();                                      // an aligned load: not every lane stored in the turn before
        tmem_ld_32x32(tmem + lanes + (unsigned)(d * acc_w + m0), v);
        if (m0 + 32 >= bn) {                               // in registers: the issuer may have the accumulator back
          tc05_fence_before_sync();
          __syncwarp();
          if (lane == 0) { if (PAIR) w4_arrive_leader(&acc_empty[d]); else mbar_arrive(&acc_empty[d]); }
        }
        if (!PAIR && parts > 1) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (m0 + j < bn) partial[(m0 + j) * 128 + (warp & 3) * 32 + lane] = v[j];
        } else {
          w4_store<TO>(out, ldo, v, m_base, m0, rows, n_base + lane, N, lane, vec2 && n_base + 32 <= N);
        }
      }
    }
  }
  if (!PAIR && parts > 1) {                                // one tile a cluster
    cluster_sync_all();                                    // every block's sums lie in its shared memory
    const int m_base = first % m_tiles * bn, n0 = first / m_tiles * 128;
    const int lo = bn * part / parts, hi = min(M - m_base, bn * (part + 1) / parts);
    const bool vec = ldo % 4 == 0 && (uintptr_t)out % 16 == 0;
    for (int i = threadIdx.x; i < (hi - lo) * 32; i += W4_THREADS) {
      const int m = lo + (i >> 5), c4 = (i & 31) * 4, n = n0 + c4;
      const float* at = partial + m * 128 + c4;
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
  __syncwarp();
  tc05_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();       // no CTA frees tensor memory the other one's instructions use
  if (warp == 3) { if (PAIR) tmem_dealloc_pair(tmem, 512); else tmem_dealloc(tmem, 512); }
}

struct W4Shape { bool pair; int bn, m_tiles, parts; };

static void w4_tc_config(cudaLaunchConfig_t* cfg, unsigned blocks, int cluster, cudaStream_t stream, cudaLaunchAttribute* attr) {
  cfg->gridDim = dim3(blocks);
  cfg->blockDim = dim3(W4_THREADS);
  cfg->dynamicSmemBytes = W4_TC_SMEM + 1024;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attr;
  cfg->numAttrs = si_pdl_enabled() ? 2 : 1;
}

// Clusters of `size` blocks that the device runs at once (the SMs of a cluster lie together, so not every one finds its place), asked once per device
// and size; all forms of the kernel take an SM a block.
static int w4_clusters(int size) {
  static int known[64][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (size == 1) return si_sm_count();
  if (!known[dev][size]) {
    auto k = gemm_w4_tc_kernel<false, true, true, bf16>;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = {};
    w4_tc_config(&cfg, (unsigned)size, size, 0, attr);
    int n = 0;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_TC_SMEM + 1024) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = 1; }
    known[dev][size] = n;
  }
  return known[dev][size];
}

// The shape for which the busiest SM is done first, in clocks: a step of 256 is bn * 8 of the tensor cores (4,096 products a clock and SM) and 200 beside them,
// 1,000 at least (widening, a wait, a commit), and for a CTA alone what taking in its bn rows of x lasts (60 bytes a clock). Where there is one accumulator its
// stores come on top. More and narrower tiles have to save a sixteenth: they cost more power, at whose cap long products run. us, the rule's choice first
// (P: two CTAs a tile, then columns and cuts of k): 16 x 4,096 x 4,096 16/4 8.2, 16/2 9.5, 16/1 13.8; 61 x 6,144 x 4,096 64/2 11.3, 64/1 15.4; 128 x
// 28,672 x 4,096 P128 32.1, 128/1 33.3; 128 x 4,096 x 14,336 128/4 20.5, 64/2 25.4; 200 x 4,096 x 14,336 112/2 28.6, P64 43.3; 300 x 4,096 x 4,096 P80 18.3,
// 80/1 17.5; 512 x 4,096 x 14,336 P128 53.1, 128/1 55.2, P176 57.6, P256 75.5; 937 x 4,096 x 14,336 P240 81, P112 100; 2,048 x 28,672 x 4,096 P256 363, P128
// 357, P192 371.
static W4Shape w4_shape(int M, int N, int K) {
  const int nk = (K + 255) / 256, fewest = (M + 255) / 256;
  W4Shape best = {false, 128, 1, 1};
  long long least = -1;
  auto consider = [&](bool pair, int bn, int mt, int parts) {
    const long long tiles = (long long)((N + (pair ? 255 : 127)) / (pair ? 256 : 128)) * mt, slots = w4_clusters(pair ? 2 : parts);
    if (parts > 1 && tiles > slots) return;
    const int steps = (nk + parts - 1) / parts;
    long long step = bn * 8 + 200;
    if (step < 1000) step = 1000;
    if (!pair && step < (16384 + bn * 512) / 60) step = (16384 + bn * 512) / 60;
    const long long cost = (tiles + slots - 1) / slots * (steps * step + (bn > 128 ? 8 * bn : 300)) + 12 * bn + (parts > 1 ? 2500 : 0);
    if (least < 0 || cost * 16 < least * 15) { least = cost; best = W4Shape{pair, bn, mt, parts}; }
  };
  for (int mt = fewest; mt <= fewest + 8; ++mt) {
    const int bn = ((M + mt - 1) / mt + 15) / 16 * 16;
    if (mt > fewest && bn < 64) break;
    if (M > 64) consider(true, bn, mt, 1);
    if (bn <= 128)                                         // a CTA alone holds 128 rows of x a slot
      for (int parts = 1; parts <= 8 && parts <= nk; parts *= 2) consider(false, bn, mt, parts);
  }
  return best;
}

template <bool PAIR, bool ZEROS, bool SMALL, typename TO>
static int w4_tc_launch(const W4Call& c, const W4Shape& sh) {
  auto k = gemm_w4_tc_kernel<PAIR, ZEROS, SMALL, TO>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_TC_SMEM + 1024);
  if (e != cudaSuccess) return (int)e;
  CUtensorMap xm, wm;
  int rc = w4_encode(&xm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, c.x, c.M, c.K, c.ldx, 64, (unsigned)(PAIR ? sh.bn / 2 : sh.bn), CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = w4_encode(&wm, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, c.w, c.N, c.K / 8, c.ldw, 16, 128, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc) return rc;
  const int cluster = PAIR ? 2 : sh.parts;
  const long long tiles = (long long)((c.N + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128)) * sh.m_tiles, slots = w4_clusters(cluster);
  if (tiles > 0x0fffffffLL) return -2;
  const long long blocks = (tiles < slots || cluster == sh.parts && cluster > 1 ? tiles : slots) * cluster;      // a tile cut over a cluster is its only one
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  w4_tc_config(&cfg, (unsigned)blocks, cluster, c.stream, attr);
  cudaLaunchKernelEx(&cfg, k, xm, wm, c.scales, c.zeros, c.group, c.groups, (TO*)c.out, c.ldo, c.M, c.N, c.K, sh.bn, sh.m_tiles, sh.parts, c.status,
                     si_pdl_trigger_mode(blocks, si_sm_count()));
  return si_last_error();
}

template <typename TO>
static int w4_tc(const W4Call& c) {
  const W4Shape sh = w4_shape(c.M, c.N, c.K);
#define W4_TC(PAIR, ZEROS) (c.group < 128 ? w4_tc_launch<PAIR, ZEROS, true, TO>(c, sh) : w4_tc_launch<PAIR, ZEROS, false, TO>(c, sh))
  if (sh.pair) return c.zeros ? W4_TC(true, true) : W4_TC(true, false);
  return c.zeros ? W4_TC(false, true) : W4_TC(false, false);
#undef W4_TC
}

// 1 when these kernels take operands so laid out (rows that start on 16-byte boundaries and end on one, the driver's tensor maps), else
// gemm_quant.cu does.
SI_EXPORT int si_gemm_w4_ok(const void* x, long long ldx, const void* w, long long ldw, int K) {
  return si_encode_fn() != nullptr && ((uintptr_t)x | (uintptr_t)w) % 16 == 0 && ldx % 8 == 0 && ldw % 4 == 0 && K % 32 == 0 && ldx >= K && ldw >= K / 8;
}

// x [M, K] bf16, rows `ldx` apart; w [N, K / 8] int32 words, rows `ldw` words apart; scales bf16 [N, ceil(K / group)], zeros uint8 like them or null;
// group 32, 64 or a multiple of 128; out [M, N], rows `ldo` apart, SI_BF16 or SI_F32. Returns 0, a CUDA error code, or -2 (size or layout refused).
static int gemm_w4(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, int group, void* out,
                         long long ldo, int out_dtype, int M, int N, int K, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 8 || K > 0x3fffffff || !(group == 32 || group == 64 || (group > 0 && group % 128 == 0)) || !si_gemm_w4_ok(x, ldx, w, ldw, K)) return -2;
  W4Call c;
  c.x = (const bf16*)x; c.ldx = ldx; c.w = (const unsigned*)w; c.ldw = ldw; c.scales = (const bf16*)scales; c.zeros = (const unsigned char*)zeros;
  c.group = group; c.groups = (K - 1) / group + 1; c.out = out; c.ldo = ldo; c.M = M; c.N = N; c.K = K; c.status = status; c.stream = stream;
  W4Few f;
  const bool wide = group >= 128 || ((uintptr_t)scales % 16 == 0 && (uintptr_t)zeros % 8 == 0);      // small groups' scales come eight at a time
  if (wide && w4_few_shape(M, N, K, zeros != nullptr, group < 128, &f)) return out_dtype == SI_BF16 ? w4_few<bf16>(c, f) : w4_few<float>(c, f);
  return out_dtype == SI_BF16 ? w4_tc<bf16>(c) : w4_tc<float>(c);
}

// The same with its arguments in one array, in their order (see quant_rows.cu).
SI_EXPORT int si_gemm_w4(const long long* a) {
  return gemm_w4((const void*)a[0], a[1], (const void*)a[2], a[3], (const void*)a[4], (const void*)a[5], (int)a[6], (void*)a[7], a[8], (int)a[9], (int)a[10],
                 (int)a[11], (int)a[12], (int*)a[13], (cudaStream_t)a[14]);
}
