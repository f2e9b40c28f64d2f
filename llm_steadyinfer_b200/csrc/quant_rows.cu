// Rows to 8 bits with a scale a row, fused with what makes them: the residual add and RMS norm, the gated activation, or nothing.
//   norm:      h = resid (+ delta (+ delta2));  dst <- h;  y = weight * h * rsqrt(mean(h^2) + eps)
//   swiglu:    y = silu(gate) * up
//   quantize:  y = x
//   scale[r] = max(max_i |y[r, i]|, 2^-100) / 448;   out[r, i] = e4m3(y[r, i] / scale[r])
// The reference has neither 8-bit type nor these kernels; the bf16 siblings are norm.cu and swiglu.cu.
//
// All three are one pass over memory: a block takes a row, every thread keeps its part of it (eight entries a load, up to 32) in
// registers over the one reduction that the row needs. The norm needs no second one: max |y| = rsqrt(...) * max |weight * h|, so the sum of
// squares and the maximum are reduced together. Arithmetic is fp32; the only rounding is the one to e4m3. Rows that are not in 16-byte
// pieces go entry by entry (us, 4,093 columns and 4,096: norm of 2,048 rows 25, 17; 4,096 rows as they are 17, 12); rows wider than 16,384 take a scalar
// kernel that reads them twice (the second time from cache).
// NaN: a NaN entry becomes a NaN code and leaves the maximum to the others (fmaxf); with an infinite entry the factor is zero and the
// entry itself becomes NaN. The norm of a row with either is NaN where the formula says so.
#include <string.h>
#include "quant_common.cuh"

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
// Eight entries as they were loaded: bf16 take half the registers of what they are widened to.
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  uint4 r;
  __device__ __forceinline__ void load(const bf16* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// The block's sum of `s` and maximum of `m`, for every thread; `scratch` holds 64 floats. Called once a kernel.
__device__ __forceinline__ float2 block_sum_max(float s, float m, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  s = warp_sum(s);
  m = warp_max(m);
  if (nwarps == 1) return make_float2(s, m);
  if (lane == 0) { scratch[warp] = s; scratch[32 + warp] = m; }
  __syncthreads();
  s = lane < nwarps ? scratch[lane] : 0.f;               // every warp adds the warps' sums up itself: no second barrier
  m = lane < nwarps ? scratch[32 + lane] : 0.f;
  return make_float2(warp_sum(s), warp_max(m));
}

struct NormArgs {
  float* resid;                 // [*, width]
  const void* delta;            // like resid, TX, or null
  const void* delta2;           // beside delta, or null
  float* dst;                   // where the stream goes, or null: it stays as it is
  const int* rows;              // row r is stream row rows[r], or null
  const void* weight;
  float eps;
  const void* ahead;            // what the next kernel streams, fetched into L2 by the blocks behind the rows
  long long ahead_bytes;
};

template <typename TX, typename TW, int CHUNKS>
__global__ void __launch_bounds__(512) norm_q8_kernel(const NormArgs a, unsigned char* out, float* scale,
                                                      int width, int num_rows, int trigger) {
  __shared__ float scratch[64];
  if (trigger) pdl_trigger();
  if ((int)blockIdx.x >= num_rows) {
    l2_prefetch_share(a.ahead, a.ahead_bytes, blockIdx.x - num_rows, gridDim.x - num_rows);
    return;
  }
  const TW* weight = (const TW*)a.weight;
  const int nchunks = width >> 3;
  if (trigger) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int ch = threadIdx.x + c * blockDim.x;
      if (ch < nchunks) prefetch_l1(weight + ch * 8);
    }
  }
  pdl_wait();
  const int r = blockIdx.x;
  const size_t src = (size_t)(a.rows ? a.rows[r] : r) * width;
  const TX* d1 = (const TX*)a.delta;
  const TX* d2 = (const TX*)a.delta2;
  float x[CHUNKS][8];
  Raw8<TX> e1[CHUNKS], e2[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = threadIdx.x + c * blockDim.x;
    if (ch < nchunks) {
      load8(a.resid + src + ch * 8, x[c]);
      if (d1) e1[c].load(d1 + src + ch * 8);
      if (d2) e2[c].load(d2 + src + ch * 8);
    }
  }
  float ss = 0.f, top = 0.f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = threadIdx.x + c * blockDim.x;
    if (ch < nchunks) {
      float e[8];
      if (d1) {
        e1[c].get(e);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] += e[i];
      }
      if (d2) {
        e2[c].get(e);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] += e[i];
      }
      if (a.dst) store8(a.dst + src + ch * 8, x[c]);
      float w[8];
      load8(weight + ch * 8, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss += x[c][i] * x[c][i];
        x[c][i] *= w[i];
        top = fmaxf(top, fabsf(x[c][i]));
      }
    }
  }
  const float2 both = block_sum_max(ss, top, scratch);
  const float inv = rsqrtf(both.x / (float)width + a.eps);
  const Q8Row to(both.y * inv);
  if (threadIdx.x == 0) scale[r] = to.scale;
  unsigned char* o = out + (size_t)r * width;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = threadIdx.x + c * blockDim.x;
    if (ch < nchunks) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] *= inv;
      *reinterpret_cast<uint2*>(o + ch * 8) = q8_pack8(to, x[c]);
    }
  }
}

// Rows that are not in 16-byte pieces: entry by entry, but in one pass as well, a thread's K in registers. (Read twice by a loop, with one entry
// under way a thread, 2,048 x 4,093 took 36 us, 4,096 x 4,093 as they are 39, 2,048 x 14,330 gated 113 for 63.)
template <typename TX, typename TW, int K>
__global__ void __launch_bounds__(1024) norm_q8_odd_kernel(const NormArgs a, unsigned char* out, float* scale, int width) {
  __shared__ float scratch[64];
  pdl_wait();
  const int r = blockIdx.x;
  const size_t src = (size_t)(a.rows ? a.rows[r] : r) * width;
  const TX* d1 = (const TX*)a.delta;
  const TX* d2 = (const TX*)a.delta2;
  const TW* weight = (const TW*)a.weight;
  float x[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const size_t i = src + min((int)(threadIdx.x + k * blockDim.x), width - 1);      // beyond the end the last entry again: no branch between the loads
    x[k] = a.resid[i];
    if (d1) x[k] += to_f32<TX>(d1[i]);
    if (d2) x[k] += to_f32<TX>(d2[i]);
  }
  float ss = 0.f, top = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < width) {
      if (a.dst) a.dst[src + i] = x[k];
      ss += x[k] * x[k];
      x[k] *= to_f32<TW>(weight[i]);
      top = fmaxf(top, fabsf(x[k]));
    }
  }
  const float2 both = block_sum_max(ss, top, scratch);
  const float inv = rsqrtf(both.x / (float)width + a.eps);
  const Q8Row to(both.y * inv);
  if (threadIdx.x == 0) scale[r] = to.scale;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < width) out[(size_t)r * width + i] = q8_pack1(to, x[k] * inv);
  }
}

template <typename TX, typename TW>
__global__ void norm_q8_scalar_kernel(const NormArgs a, unsigned char* out, float* scale, int width) {
  __shared__ float scratch[64];
  pdl_wait();
  const int r = blockIdx.x;
  const size_t src = (size_t)(a.rows ? a.rows[r] : r) * width;
  const TX* d1 = (const TX*)a.delta;
  const TX* d2 = (const TX*)a.delta2;
  const TW* weight = (const TW*)a.weight;
  auto entry = [&](int i) {
    float h = a.resid[src + i];
    if (d1) h += to_f32<TX>(d1[src + i]);
    if (d2) h += to_f32<TX>(d2[src + i]);
    return h;
  };
  float ss = 0.f, top = 0.f;
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    const float h = entry(i);
    if (a.dst) a.dst[src + i] = h;
    ss += h * h;
    top = fmaxf(top, fabsf(h * to_f32<TW>(weight[i])));
  }
  const float2 both = block_sum_max(ss, top, scratch);
  const float inv = rsqrtf(both.x / (float)width + a.eps);
  const Q8Row to(both.y * inv);
  if (threadIdx.x == 0) scale[r] = to.scale;
  for (int i = threadIdx.x; i < width; i += blockDim.x) {            // what this thread stored itself, where the stream was written
    const float h = a.dst ? a.dst[src + i] : entry(i);
    out[(size_t)r * width + i] = q8_pack1(to, h * to_f32<TW>(weight[i]) * inv);
  }
}

// silu(g) * u with the hardware's exponential of base 2 and reciprocal: off by 2 + 1.2 |g| units where g is negative (and exp(-g) large), by four where it
// is positive. The reciprocal is that of a quarter of 1 + exp(-g), which it can take up to 2^126 without a subnormal result, and u the other quarter: so all
// gates down to -88.7, where exp(-g) passes fp32's range and the result is zero, are as the formula has them. (ftz changes exp(-g) alone, where it is nothing
// beside one.) Two entries at a time. With the accurate functions arithmetic bounded the kernel: 84 us for 2,048 x 14,336, the accurate quotient alone 50 of them.
__device__ __forceinline__ void silu_mul_q8(float& g0, float& g1, float u0, float u1) {
  asm("{\n.reg .f32 a, b;\n.reg .b64 g, e, c;\n"
      "mov.b64 g, {%0, %1};\nmov.b64 c, {%4, %4};\nmul.rn.f32x2 e, g, c;\n"
      "mov.b64 {a, b}, e;\nex2.approx.ftz.f32 a, a;\nex2.approx.ftz.f32 b, b;\nmov.b64 e, {a, b};\n"
      "mov.b64 c, {%5, %5};\nfma.rn.f32x2 e, e, c, c;\n"
      "mov.b64 {a, b}, e;\nrcp.approx.ftz.f32 a, a;\nrcp.approx.ftz.f32 b, b;\nmov.b64 e, {a, b};\n"
      "mul.rn.f32x2 g, g, e;\nmov.b64 e, {%2, %3};\nmul.rn.f32x2 e, e, c;\nmul.rn.f32x2 g, g, e;\nmov.b64 {%0, %1}, g;\n}\n"
      : "+f"(g0), "+f"(g1) : "f"(u0), "f"(u1), "f"(-1.4426950408889634f), "f"(0.25f));
}
__device__ __forceinline__ float silu_mul_q8(float g, float u) {
  float e, q;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(__fmaf_rn(e, 0.25f, 0.25f)));
  return g * q * (u * 0.25f);
}

// x as it is: the loaded entries stay packed in registers and are widened twice, before and after the reduction. A block goes through rows, and asks for
// its next one before it reduces this one.
template <typename TX, int CHUNKS>
__global__ void __launch_bounds__(512, sizeof(TX) == 2 || CHUNKS < 4 ? 2 : 1)
rows_q8_kernel(const TX* x, long long ldx, unsigned char* out, float* scale, int width, int num_rows, int trigger) {
  __shared__ float scratch[2][64];
  if (trigger) pdl_trigger();
  pdl_wait();
  const int nchunks = width >> 3;
  Raw8<TX> raw[CHUNKS], next[CHUNKS];
  auto load = [&](int r, Raw8<TX> (&to)[CHUNKS]) {
    const TX* row = x + (size_t)r * ldx;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int ch = threadIdx.x + c * blockDim.x;
      if (ch < nchunks) to[c].load(row + ch * 8);
    }
  };
  load(blockIdx.x, next);
  int par = 0;
  for (int r = blockIdx.x; r < num_rows; r += gridDim.x, par ^= 1) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) raw[c] = next[c];
    if (r + (int)gridDim.x < num_rows) load(r + gridDim.x, next);
    float top = 0.f, v[8];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if ((int)(threadIdx.x + c * blockDim.x) < nchunks) {
        raw[c].get(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
      }
    top = block_sum_max(0.f, top, scratch[par]).y;      // a buffer is written again two rows later, behind the next row's barrier
    const Q8Row to(top);
    if (threadIdx.x == 0) scale[r] = to.scale;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int ch = threadIdx.x + c * blockDim.x;
      if (ch < nchunks) {
        raw[c].get(v);
        *reinterpret_cast<uint2*>(out + (size_t)r * width + ch * 8) = q8_pack8(to, v);
      }
    }
  }
}

// The gated activation: gate f in column (f / group) * 2 * group + f % group, its up `group` columns further.
// `shift`: group's logarithm, 31 where a row is one group, or -1 where it is no power of two: a division for every eight entries was a tenth to a quarter of the whole (2,048 x 14,336
// 31.0 us with it and 28.2 without, 5.2 TB/s; 2,048 x 8,192 20.1 and 15.5).
template <typename TX, int CHUNKS>
__global__ void __launch_bounds__(512, CHUNKS <= 2 && sizeof(TX) == 2 ? 3 : 2) gated_q8_kernel(const TX* gu, unsigned char* out, float* scale, int width, int group, int shift,
                                                                   int trigger) {
  __shared__ float scratch[64];
  if (trigger) pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x, nchunks = width >> 3;
  const TX* row = gu + (size_t)r * 2 * width;
  Raw8<TX> gate[CHUNKS], up[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = threadIdx.x + c * blockDim.x;
    if (ch < nchunks) {
      const int f = ch * 8, at = (shift >= 0 ? f >> shift << shift : f / group * group) + f;              // (f / group) * 2 * group + f % group
      gate[c].load(row + at);
      up[c].load(row + at + group);
    }
  }
  float top = 0.f, v[CHUNKS][8];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    if ((int)(threadIdx.x + c * blockDim.x) < nchunks) {
      float u[8];
      gate[c].get(v[c]);
      up[c].get(u);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        silu_mul_q8(v[c][i], v[c][i + 1], u[i], u[i + 1]);
        top = fmaxf(top, fmaxf(fabsf(v[c][i]), fabsf(v[c][i + 1])));
      }
    }
  top = block_sum_max(0.f, top, scratch).y;
  const Q8Row to(top);
  if (threadIdx.x == 0) scale[r] = to.scale;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = threadIdx.x + c * blockDim.x;
    if (ch < nchunks) {
      *reinterpret_cast<uint2*>(out + (size_t)r * width + ch * 8) = q8_pack8(to, v[c]);
    }
  }
}

template <typename TX, bool GATED, int K>
__global__ void __launch_bounds__(1024) rows_q8_odd_kernel(const TX* x, long long ldx, unsigned char* out, float* scale, int width, int group, int shift) {
  __shared__ float scratch[64];
  pdl_wait();
  const TX* row = x + (size_t)blockIdx.x * ldx;
  float v[K], top = 0.f;
#pragma unroll
  for (int b = 0; b < K; b += 8) {                        // eight at a time: sixteen gates and ups with their addresses are more than a thread's registers
    float up[GATED ? 8 : 1];
#pragma unroll
    for (int k = 0; k < 8; ++k) {                         // beyond the end the last entry again: no branch between the loads, no other maximum
      const int i = min((int)(threadIdx.x + (b + k) * blockDim.x), width - 1);
      const int at = !GATED ? i : (shift >= 0 ? i >> shift << shift : i / group * group) + i;
      v[b + k] = to_f32<TX>(row[at]);
      if (GATED) up[k] = to_f32<TX>(row[at + group]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (GATED) v[b + k] = silu_mul_q8(v[b + k], up[k]);
      top = fmaxf(top, fabsf(v[b + k]));
    }
    if (GATED) asm volatile("" ::: "memory");
  }
  top = block_sum_max(0.f, top, scratch).y;
  const Q8Row to(top);
  if (threadIdx.x == 0) scale[blockIdx.x] = to.scale;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < width) out[(size_t)blockIdx.x * width + i] = q8_pack1(to, v[k]);
  }
}

template <typename TX, bool GATED>
__global__ void rows_q8_scalar_kernel(const TX* x, long long ldx, unsigned char* out,
                                      float* scale, int width, int group) {
  __shared__ float scratch[64];
  pdl_wait();
  const TX* row = x + (size_t)blockIdx.x * ldx;
  auto entry = [&](int i) {
    if (!GATED) return to_f32<TX>(row[i]);
    const int at = i / group * group + i;
    return silu_mul_q8(to_f32<TX>(row[at]), to_f32<TX>(row[at + group]));
  };
  float top = 0.f;
  for (int i = threadIdx.x; i < width; i += blockDim.x) top = fmaxf(top, fabsf(entry(i)));
  top = block_sum_max(0.f, top, scratch).y;
  const Q8Row to(top);
  if (threadIdx.x == 0) scale[blockIdx.x] = to.scale;
  for (int i = threadIdx.x; i < width; i += blockDim.x) out[(size_t)blockIdx.x * width + i] = q8_pack1(to, entry(i));
}

#define Q8_MAX_VEC_WIDTH (4 * 8 * 512)
// Threads of a row's block: what covers it in one load each, up to 512; then two or four loads each.
// Many rows of a norm go by half as many threads with twice the loads each, so that more blocks, in different phases, share an SM.
static int row_threads(int width, int most = 512) {
  const int chunks = (width + 7) / 8;
  return chunks >= most ? most : (chunks + 31) / 32 * 32;
}

static dim3 odd_threads(int width, int each) { return dim3(((width + each - 1) / each + 31) / 32 * 32); }

template <typename TX, typename TW>
static void launch_norm(const NormArgs& a, unsigned char* out, float* scale, int width, int num_rows, bool vec, cudaStream_t stream) {
  const dim3 block(row_threads(width, vec && num_rows >= 1024 && width <= Q8_MAX_VEC_WIDTH / 2 ? 256 : 512));
  if (!vec) {
#define NORM_ODD(K) si_launch(norm_q8_odd_kernel<TX, TW, K>, dim3(num_rows), odd_threads(width, K), 0, stream, a, out, scale, width)
    if (width <= 8 * 1024) NORM_ODD(8);
    else if (width <= 16 * 1024) NORM_ODD(16);
    else si_launch(norm_q8_scalar_kernel<TX, TW>, dim3(num_rows), block, 0, stream, a, out, scale, width);
#undef NORM_ODD
    return;
  }
  const int per = (width / 8 + block.x - 1) / block.x, sms = si_sm_count();
  const int trigger = si_pdl_trigger_enabled() && num_rows <= 64;
  const int extra = a.ahead ? (num_rows < sms ? 2 * sms - num_rows : sms) : 0;
  const dim3 grid(num_rows + extra);
#define NORM_Q8(C) si_launch(norm_q8_kernel<TX, TW, C>, grid, block, 0, stream, a, out, scale, width, num_rows, trigger)
  if (per <= 1) NORM_Q8(1); else if (per <= 2) NORM_Q8(2); else NORM_Q8(4);
#undef NORM_Q8
}

// resid [*, width] fp32; delta, delta2 (may be null) like it in x_dtype; weight [width] in w_dtype; dst (may be null, may be resid);
// out [num_rows, width] e4m3, scale [num_rows] fp32. Returns 0, a CUDA error code, or -2 (size refused).
static int add_rmsnorm_q8(float* resid, const void* delta, const void* delta2, int x_dtype, const int* rows, const void* weight,
                                int w_dtype, float* dst, void* out, float* scale, int num_rows, int width, float eps, const void* ahead,
                                long long ahead_bytes, cudaStream_t stream) {
  if (num_rows <= 0) return 0;
  if (width <= 0 || (delta2 && !delta)) return -2;
  NormArgs a;
  a.resid = resid; a.delta = delta; a.delta2 = delta2; a.dst = dst; a.rows = rows; a.weight = weight; a.eps = eps;
  a.ahead = ahead_bytes >= 4096 ? ahead : nullptr; a.ahead_bytes = ahead_bytes;
  const bool vec = width % 8 == 0 && width <= Q8_MAX_VEC_WIDTH &&
                   (((uintptr_t)resid | (uintptr_t)delta | (uintptr_t)delta2 | (uintptr_t)dst | (uintptr_t)weight) % 16 == 0) && (uintptr_t)out % 8 == 0;
  unsigned char* o = (unsigned char*)out;
  if (x_dtype == SI_BF16) {
    if (w_dtype == SI_BF16) launch_norm<bf16, bf16>(a, o, scale, width, num_rows, vec, stream);
    else launch_norm<bf16, float>(a, o, scale, width, num_rows, vec, stream);
  } else {
    if (w_dtype == SI_BF16) launch_norm<float, bf16>(a, o, scale, width, num_rows, vec, stream);
    else launch_norm<float, float>(a, o, scale, width, num_rows, vec, stream);
  }
  return si_last_error();
}

template <typename TX, bool GATED>
static void launch_rows(const void* x, long long ldx, void* out, float* scale, int num_rows, int width, int group, cudaStream_t stream) {
  dim3 grid(num_rows), block(row_threads(width));
  const TX* xp = (const TX*)x;
  unsigned char* o = (unsigned char*)out;
  const bool vec = width % 8 == 0 && width <= Q8_MAX_VEC_WIDTH && (!GATED || group % 8 == 0) && ldx % (16 / (int)sizeof(TX)) == 0 &&
                   (uintptr_t)x % 16 == 0 && (uintptr_t)out % 8 == 0;
  const int shift = group >= width ? 31 : (group & (group - 1)) == 0 ? __builtin_ctz(group) : -1;      // one group: 31, nothing is left of a column
  if (!vec) {
#define ROWS_ODD(K) si_launch(rows_q8_odd_kernel<TX, GATED, K>, grid, odd_threads(width, K), 0, stream, xp, ldx, o, scale, width, group, shift)
    if (width <= 8 * 1024) ROWS_ODD(8);
    else if (width <= 16 * 1024) ROWS_ODD(16);
    else si_launch(rows_q8_scalar_kernel<TX, GATED>, grid, block, 0, stream, xp, ldx, o, scale, width, group);
#undef ROWS_ODD
    return;
  }
  const int least = (width / 8 + block.x - 1) / block.x, per = least <= 2 ? least : 4, trigger = si_pdl_trigger_small(num_rows);
  block.x = ((width / 8 + per - 1) / per + 31) / 32 * 32;           // no more than have work: 2,048 x 5,632 gated 12.8 us with 512 threads, 11.1 with 352
  const int most = si_sm_count() * (int)(1024 / block.x);          // blocks that run at once
  if (!GATED && num_rows > most) grid.x = most;
#define ROWS_Q8(C) do { if constexpr (GATED) si_launch(gated_q8_kernel<TX, C>, grid, block, 0, stream, xp, o, scale, width, group, shift, trigger); \
                        else si_launch(rows_q8_kernel<TX, C>, grid, block, 0, stream, xp, ldx, o, scale, width, num_rows, trigger); } while (0)
  if (per == 1) ROWS_Q8(1); else if (per == 2) ROWS_Q8(2); else ROWS_Q8(4);
#undef ROWS_Q8
}

// x [num_rows, width], rows `ldx` entries apart -> out [num_rows, width] e4m3, scale [num_rows].
static int quantize_q8(const void* x, int dtype, long long ldx, void* out, float* scale, int num_rows, int width, cudaStream_t stream) {
  if (num_rows <= 0) return 0;
  if (width <= 0) return -2;
  if (dtype == SI_BF16) launch_rows<bf16, false>(x, ldx, out, scale, num_rows, width, 1, stream);
  else launch_rows<float, false>(x, ldx, out, scale, num_rows, width, 1, stream);
  return si_last_error();
}

// gu [num_rows, 2 * inter], rows one behind the other, gates and ups interleaved in groups of `group` columns -> out [num_rows, inter].
static int swiglu_q8(const void* gu, int dtype, void* out, float* scale, int num_rows, int inter, int group, cudaStream_t stream) {
  if (num_rows <= 0) return 0;
  if (inter <= 0 || group <= 0 || inter % group || inter > 0x3fffffff) return -2;
  if (dtype == SI_BF16) launch_rows<bf16, true>(gu, 2LL * inter, out, scale, num_rows, inter, group, stream);
  else launch_rows<float, true>(gu, 2LL * inter, out, scale, num_rows, inter, group, stream);
  return si_last_error();
}

// The functions above with their arguments in one array, in their order (eps as a double): handing over up to sixteen one by one cost the calling side
// 2.3 us, an array 0.6.
SI_EXPORT int si_add_rmsnorm_q8(const long long* a) {
  double eps;
  memcpy(&eps, a + 12, 8);
  return add_rmsnorm_q8((float*)a[0], (const void*)a[1], (const void*)a[2], (int)a[3], (const int*)a[4], (const void*)a[5], (int)a[6], (float*)a[7],
                        (void*)a[8], (float*)a[9], (int)a[10], (int)a[11], (float)eps, (const void*)a[13], a[14], (cudaStream_t)a[15]);
}
SI_EXPORT int si_quantize_q8(const long long* a) {
  return quantize_q8((const void*)a[0], (int)a[1], a[2], (void*)a[3], (float*)a[4], (int)a[5], (int)a[6], (cudaStream_t)a[7]);
}
SI_EXPORT int si_swiglu_q8(const long long* a) {
  return swiglu_q8((const void*)a[0], (int)a[1], (void*)a[2], (float*)a[3], (int)a[4], (int)a[5], (int)a[6], (cudaStream_t)a[7]);
}
