// Products with quantised operands, for any size, stride and alignment:
//   8 bits:  out[m, n] = sa[m] * sw[n] * sum_k a[m, k] w[n, k]          a, w e4m3, scales fp32
//   4 bits:  out[m, n] = sum_k x[m, k] * s[n, k / group] * (q[n, k] - z[n, k / group])      x bf16
// This is the form that takes what the fast kernels (gemm_q8.cu, gemm_w4.cu) do not: rows that are not in 16-byte pieces.
//
// Tiles of 64 rows of x by 128 output columns, eight warps as 2 x 4, 32-wide k steps through two buffers of shared memory; the next step's
// operands are on their way to registers while mma.sync runs on this one's. The operands are widened on the way to shared memory to a type that
// holds every value exactly: e4m3 to fp16 (its range and its three mantissa bits fit), bf16 stays. A 4-bit weight times its scale is rounded
// to bf16 there (off by at most 2^-8 of its value) whatever the number of rows, as gemm_w4.cu does for many. Sums are fp32. Rows of 32 entries lie 80 bytes apart:
// ldmatrix's eight rows then fall into different banks.
//
// Where tiles are fewer than blocks that run at once, the k steps of one are shared by the blocks of a cluster; each leaves its sums in its shared memory
// and adds a part of the rows up over all blocks, in their order (us with one block a tile and so: 8 bits 8 x 4,000 x 4,088 137, 25; 61 x 500 x 7,000 236, 35;
// 4 bits 212, 37 and 303, 45; the first of them with rows of w on no 8-byte boundary, whose bytes come one by one, 45 to 55).
#include "tma_common.cuh"
#include "quant_common.cuh"

typedef __nv_bfloat16 bf16;

constexpr int GQ_BM = 64, GQ_BN = 128, GQ_BK = 32, GQ_LD = 40;      // GQ_LD: entries between rows in shared memory

__device__ __forceinline__ unsigned gq_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void gq_ldmatrix4(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool HALF>
__device__ __forceinline__ void gq_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  if (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// BYTES bytes of a row from byte `k` on (the row is `len` bytes), in 4-byte words: beyond the end zeros. `wide`: the row starts at a multiple
// of BYTES, or of 8 where BYTES is 16.
template <int BYTES>
__device__ __forceinline__ void gq_load(const unsigned char* row, int k, int len, bool wide, unsigned (&v)[BYTES / 4]) {
  if (wide && k + BYTES <= len) {
#pragma unroll
    for (int i = 0; i < BYTES / 8; ++i) {
      const uint2 t = *reinterpret_cast<const uint2*>(row + k + 8 * i);
      v[2 * i] = t.x; v[2 * i + 1] = t.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < BYTES / 4; ++i) {
    unsigned w = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (k + 4 * i + b < len) w |= (unsigned)row[k + 4 * i + b] << (8 * b);
    v[i] = w;
  }
}

__device__ __forceinline__ float gq_ld_cluster(unsigned cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

struct QuantProduct {
  const void* x; long long ldx;           // e4m3 or bf16, entries between rows
  const void* w; long long ldw;           // e4m3 (entries) or int32 words of eight entries (words)
  const float* x_scale; const float* w_scale;                                   // 8 bits
  const bf16* scales; const unsigned char* zeros; int group, groups;             // 4 bits: [N, groups]
  int M, N, K;
  bool wide_x, wide_w;                    // rows start on 8-byte boundaries
};

template <bool W4, typename TO>
__global__ void __launch_bounds__(256) gemm_quant_kernel(const QuantProduct p, TO* out, long long ldo, int n_tiles, int parts) {
  __shared__ __align__(16) unsigned char raw[GQ_BM * GQ_BN * 4];              // two buffers of both operands, then the block's sums
  unsigned short (*As)[GQ_BM * GQ_LD] = reinterpret_cast<unsigned short (*)[GQ_BM * GQ_LD]>(raw);
  unsigned short (*Bs)[GQ_BN * GQ_LD] = reinterpret_cast<unsigned short (*)[GQ_BN * GQ_LD]>(raw + 2 * sizeof(*As));
  static_assert(2 * (sizeof(*As) + sizeof(*Bs)) <= sizeof(raw), "the operands fit");
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = (int)(blockIdx.x / parts), part = parts > 1 ? (int)cluster_cta_rank() : 0;
  const int m0 = tile / n_tiles * GQ_BM, n0 = tile % n_tiles * GQ_BN;
  // who fetches what of a step: eight entries of a row of x, sixteen of a row of W
  const int am = tid >> 2, ak = (tid & 3) * 8, bn = tid >> 1, bk = (tid & 1) * 16;
  const bool a_in = m0 + am < p.M, b_in = n0 + bn < p.N;
  constexpr int A_BYTES = W4 ? 16 : 8, B_BYTES = W4 ? 8 : 16, A_SIZE = W4 ? 2 : 1;
  const unsigned char* arow = (const unsigned char*)p.x + (size_t)(a_in ? m0 + am : 0) * p.ldx * A_SIZE;
  const unsigned char* brow = (const unsigned char*)p.w + (size_t)(b_in ? n0 + bn : 0) * p.ldw * (W4 ? 4 : 1);
  const int a_len = a_in ? p.K * A_SIZE : 0, b_len = b_in ? (W4 ? p.K / 2 : p.K) : 0;      // 4 bits: K is a multiple of 8
  unsigned av[A_BYTES / 4], bv[B_BYTES / 4];
  float s = 0.f;
  int z = 8;
  auto fetch = [&](int k0) {
    gq_load<A_BYTES>(arow, (k0 + ak) * A_SIZE, a_len, p.wide_x, av);
    gq_load<B_BYTES>(brow, W4 ? (k0 + bk) / 2 : k0 + bk, b_len, p.wide_w, bv);
    if (W4 && b_in && k0 + bk < p.K) {                                     // a step of 32 lies in one group
      const size_t g = (size_t)(n0 + bn) * p.groups + (k0 + bk) / p.group;
      s = __bfloat162float(p.scales[g]);
      z = p.zeros ? (int)p.zeros[g] : 8;
    }
  };
  auto widen = [](unsigned v, unsigned* to) {                              // four e4m3 -> two pairs of fp16
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> (16 * h)), __NV_E4M3);
      to[h] = (unsigned)r.x | ((unsigned)r.y << 16);
    }
  };
  auto put = [&](int buf, int k0) {
    unsigned* a = reinterpret_cast<unsigned*>(&As[buf][am * GQ_LD + ak]);
    unsigned* b = reinterpret_cast<unsigned*>(&Bs[buf][bn * GQ_LD + bk]);
    if constexpr (W4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = av[i];
      const __nv_bfloat162 bias = w4_bias(z), sc = __float2bfloat162_rn(s);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const unsigned v = w4_pair(bv[i], q, bias);
          const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), sc);
          b[4 * i + q] = b_in && k0 + bk + 8 * i < p.K ? *reinterpret_cast<const unsigned*>(&r) : 0u;      // beyond the end nothing, whatever the scale is
        }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) widen(av[i], a + 2 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i) widen(bv[i], b + 2 * i);
    }
  };
  float acc[2][4][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
  const int wm = (warp >> 2) * 32, wn = (warp & 3) * 32;
  const int all = (p.K + GQ_BK - 1) / GQ_BK, first = (int)((long long)all * part / parts), steps = (int)((long long)all * (part + 1) / parts);
  fetch(first * GQ_BK);
  put(0, first * GQ_BK);
  __syncthreads();
  for (int st = first; st < steps; ++st) {
    const int buf = (st - first) & 1;
    if (st + 1 < steps) fetch((st + 1) * GQ_BK);
#pragma unroll
    for (int kk = 0; kk < GQ_BK; kk += 16) {
      unsigned a[2][4], b[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) gq_ldmatrix4(a[i], gq_smem(&As[buf][(wm + i * 16 + (lane & 15)) * GQ_LD + kk + (lane >> 4) * 8]));
#pragma unroll
      for (int j = 0; j < 2; ++j)             // matrices: columns j*16 .. +7 of k 0-7, of k 8-15, then columns j*16+8 .. of both
        gq_ldmatrix4(b[j], gq_smem(&Bs[buf][(wn + j * 16 + (lane & 7) + ((lane >> 4) << 3)) * GQ_LD + kk + ((lane >> 3) & 1) * 8]));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) gq_mma<!W4>(acc[i][j], a[i], b[j >> 1][(j & 1) * 2], b[j >> 1][(j & 1) * 2 + 1]);
    }
    if (st + 1 < steps) put(buf ^ 1, (st + 1) * GQ_BK);       // the other buffer: all warps left it before the last barrier
    __syncthreads();
  }
  if (parts > 1) {
    float* sums = reinterpret_cast<float*>(raw);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[(wm + i * 16 + (lane >> 2) + (e >> 1) * 8) * GQ_BN + wn + j * 8 + (lane & 3) * 2 + (e & 1)] = acc[i][j][e];
    cluster_sync_all();                                       // every block's sums lie in its shared memory
    const int lo = GQ_BM * part / parts, rows = GQ_BM / parts;
    for (int i = tid; i < rows * GQ_BN; i += 256) {
      const int m = m0 + lo + i / GQ_BN, n = n0 + i % GQ_BN;
      const float* at = sums + lo * GQ_BN + i;
      float t[8], v;
#pragma unroll
      for (int c = 0; c < 8; ++c) t[c] = c < parts ? gq_ld_cluster(cluster_map_u32(at, (unsigned)c)) : 0.f;
      v = t[0];
#pragma unroll
      for (int c = 1; c < 8; ++c) v += t[c];
      if (m < p.M && n < p.N) {
        if (!W4) v = q8_scaled(v, p.x_scale[m], p.w_scale[n]);
        out[(size_t)m * ldo + n] = from_f32<TO>(v);
      }
    }
    cluster_sync_all();                                       // no block goes while another one reads its sums
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + wm + i * 16 + (lane >> 2) + (e >> 1) * 8, n = n0 + wn + j * 8 + (lane & 3) * 2 + (e & 1);
        if (m < p.M && n < p.N) {
          float v = acc[i][j][e];
          if (!W4) v = q8_scaled(v, p.x_scale[m], p.w_scale[n]);
          out[(size_t)m * ldo + n] = from_f32<TO>(v);
        }
      }
}

template <bool W4>
static int gq_launch(const QuantProduct& p, void* out, long long ldo, int out_dtype, cudaStream_t stream) {
  const long long n_tiles = (p.N + GQ_BN - 1) / GQ_BN, tiles = n_tiles * ((p.M + GQ_BM - 1) / GQ_BM);
  if (tiles > 0x0fffffffLL) return -2;
  int parts = 1;                                               // two blocks an SM, eight steps a block at least
  while (parts < 8 && tiles * parts * 2 <= 2 * si_sm_count() && (p.K + GQ_BK - 1) / GQ_BK >= 16 * parts) parts *= 2;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * parts));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = si_pdl_enabled() ? 2 : 1;
  if (out_dtype == SI_BF16) cudaLaunchKernelEx(&cfg, gemm_quant_kernel<W4, bf16>, p, (bf16*)out, ldo, (int)n_tiles, parts);
  else cudaLaunchKernelEx(&cfg, gemm_quant_kernel<W4, float>, p, (float*)out, ldo, (int)n_tiles, parts);
  return si_last_error();
}

// a [M, K] and w [N, K] e4m3, rows `lda` and `ldw` apart; x_scale [M], w_scale [N] fp32; out [M, N] rows `ldo` apart, SI_BF16 or SI_F32.
SI_EXPORT int si_gemm_quant_q8(const void* a, long long lda, const float* x_scale, const void* w, long long ldw, const float* w_scale,
                               void* out, long long ldo, int out_dtype, int M, int N, int K, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 0x3fffffff) return -2;
  QuantProduct p = {};
  p.x = a; p.ldx = lda; p.x_scale = x_scale; p.w = w; p.ldw = ldw; p.w_scale = w_scale; p.M = M; p.N = N; p.K = K;
  p.wide_x = lda % 8 == 0 && (uintptr_t)a % 8 == 0;
  p.wide_w = ldw % 8 == 0 && (uintptr_t)w % 8 == 0;
  return gq_launch<false>(p, out, ldo, out_dtype, stream);
}

// x [M, K] bf16; w [N, K / 8] int32 words, rows `ldw` words apart; scales bf16 [N, ceil(K / group)], zeros uint8 like them or null (8);
// K a multiple of 8, group of 32. (K up to 2^30 - 32: the end of a row's last step of 32 entries, in bytes, has to stay below 2^31, or the check of a load
// against the row's end turns around.)
SI_EXPORT int si_gemm_quant_w4(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, int group,
                               void* out, long long ldo, int out_dtype, int M, int N, int K, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 8 || K > 0x3fffffe0 || group <= 0 || group % 32) return -2;
  QuantProduct p = {};
  p.x = x; p.ldx = ldx; p.w = w; p.ldw = ldw; p.scales = (const bf16*)scales; p.zeros = (const unsigned char*)zeros;
  p.group = group; p.groups = (K - 1) / group + 1; p.M = M; p.N = N; p.K = K;
  p.wide_x = ldx % 4 == 0 && (uintptr_t)x % 8 == 0;
  p.wide_w = ldw % 2 == 0 && (uintptr_t)w % 8 == 0;
  return gq_launch<true>(p, out, ldo, out_dtype, stream);
}
