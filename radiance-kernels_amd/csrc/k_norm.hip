// RMS norm with the residual's addition and MX E4M3 output.
#pragma once

#include "k_kv4.hip"

// h = x + residual (rounded to their type; without a residual h is x), y = h / sqrt(mean(h^2) + eps) * (w +
// w_offset) in fp32, y to E4M3 codes and E8M0 scales of rule R1, 32-blocks along the row.  The norm is that
// of the h that is stored, so whoever reads h sees what was normed.  One workgroup per row; a thread
// holds 8 consecutive elements (a quarter of a block) of up to NORM_J chunks 2,048 apart in registers between
// the sum and the output, and reads the chunks of a longer row again.  Bound by memory and, nearly as long, by
// the arithmetic of the codes: 8,192 rows of 4,096 in bf16 with a residual, 236 MB in 48 us (4.9 TB/s; a copy 5.1; 45 with y
// rounded on the way, which gave some rows codes and now and then a block's scale that are not the exact y's); 64
// rows 4.8 us, the latency of two trips to memory and a launch.
constexpr int NORM_J = 4;

template <bool F32>
__device__ __forceinline__ void norm_store8(void* base, int64_t off, const float (&x)[8]) {
  if constexpr (F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + off);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    v4i w;
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (int)pack_bf16(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<v4i*>(static_cast<uint16_t*>(base) + off) = w;
  }
}

// y g + c for |c| well below |y g|, rounded to odd: towards 0, and the last bit set if anything was cut.  A second
// rounding to few bits, and a comparison with a power of two, then come out as for the exact value.
__device__ __forceinline__ float norm_odd(float y, float g, float c) {
  const float t = __builtin_fmaf(y, g, c), r = __builtin_fmaf(y, g, -t) + c;
  const uint32_t b = __float_as_uint(t), cut = (b - ((__float_as_uint(r) ^ b) >> 31)) | 1u;
  return __builtin_amdgcn_classf(r, 0x198) && t != 0.0f ? __uint_as_float(cut) : t;   // (r finite and not 0)
}

template <bool F32>
__device__ __forceinline__ void norm_quant_impl(const NormArgs& a) {
  __shared__ double ssum[4];
  const int tid = threadIdx.x, nchunk = a.cols / 8;
  const int64_t row = blockIdx.x, base = row * a.cols;
  auto load_h = [&](float (&h)[8], int c) {
    kv4_load8<F32>(h, a.x, base + 8 * c);
    if (a.residual) {
      float r[8];
      kv4_load8<F32>(r, a.residual, base + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; i++) h[i] = F32 ? h[i] + r[i] : (float)(__bf16)(h[i] + r[i]);
    }
  };
  float h[NORM_J][8], ss = 0.0f;
#pragma unroll
  for (int j = 0; j < NORM_J; j++) {
    const int c = tid + 256 * j;
    if (c < nchunk) {
      load_h(h[j], c);
#pragma unroll
      for (int i = 0; i < 8; i++) ss = __builtin_fmaf(h[j][i], h[j][i], ss);
    }
  }
  for (int c = tid + 256 * NORM_J; c < nchunk; c += 256) {
    float t[8];
    load_h(t, c);
#pragma unroll
    for (int i = 0; i < 8; i++) ss = __builtin_fmaf(t[i], t[i], ss);
  }
  // From here to y the arithmetic is that of 64 bits (sum of the threads' sums, root, and the product, with the low parts
  // kept), and y is rounded once.
  double sum = ss;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
  if ((tid & 63) == 0) ssum[tid >> 6] = sum;
  __syncthreads();
  const double root = 1.0 / __builtin_sqrt((ssum[0] + ssum[1] + ssum[2] + ssum[3]) / a.cols + (double)a.eps);
  const float inv = (float)root, inv_lo = inv < INFINITY ? (float)(root - inv) : 0.0f;
  auto put = [&](float (&t)[8], int c) {
    if (a.h) norm_store8<F32>(a.h, base + 8 * c, t);
    float w[8], m = 0.0f;
    kv4_load8<F32>(w, a.w, 8 * c);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float y = t[i] * inv, lo = __builtin_fmaf(t[i], inv, -y) + t[i] * inv_lo, g = w[i] + a.w_offset;
      t[i] = norm_odd(y, g, lo * g);
      m = fmaxf(m, fabsf(t[i]));
    }
    const uint32_t sc = scale_code(max4(m), 8);
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = __builtin_ldexpf(t[i], 127 - (int)sc);
    const uint2 codes = make_uint2(e4m3_code4(t[0], t[1], t[2], t[3]), e4m3_code4(t[4], t[5], t[6], t[7]));
    *reinterpret_cast<uint2*>(a.codes + base + 8 * c) = codes;
    if ((c & 3) == 0) a.scales[a.sc_ld ? (c >> 2) * a.sc_ld + row : row * (a.cols / 32) + (c >> 2)] = (uint8_t)sc;
  };
#pragma unroll
  for (int j = 0; j < NORM_J; j++) {
    const int c = tid + 256 * j;
    if (c < nchunk) put(h[j], c);
  }
  for (int c = tid + 256 * NORM_J; c < nchunk; c += 256) {
    float t[8];
    load_h(t, c);
    put(t, c);
  }
}

extern "C" __global__ void __launch_bounds__(256) mxfa_rmsnorm_quant_f32(NormArgs a) { norm_quant_impl<true>(a); }
extern "C" __global__ void __launch_bounds__(256) mxfa_rmsnorm_quant_bf16(NormArgs a) { norm_quant_impl<false>(a); }
