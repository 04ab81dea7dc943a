// 4-bit KV cache: append (quantize as written), read-back, attention over it.
//
// K and V are E2M1 codes in MX blocks of 32 along the head dimension of one token, so a token is
// quantized by itself: it can be written at any position, again, and for each sequence at its own.
//   codes  [B][Hkv][L][D/2]             element 2i in the low four bits of byte i, 2i + 1 in the high
//   scales [B][Hkv][L/32][4][D/32][8]   token t of its 32 at [t % 4][block][2 (t / 4 % 4) + t / 16]
// The scales lie in the order in which the attention reads them: a lane of the PV product holds the 8
// tokens t = k (mod 4) of 32 for one block (kv4_attn_impl), whose scales are then 8 contiguous bytes.
#pragma once

#include "k_attn_common.hip"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// Byte of token t, block b of nb in a (batch, KV head)'s scales.
__device__ __forceinline__ int64_t kv4_scale_at(int t, int b, int nb) {
  return (int64_t)(t >> 5) * (32 * nb) + ((t & 3) * nb + b) * 8 + 2 * ((t >> 2) & 3) + ((t >> 4) & 1);
}

// Maximum over aligned groups of 4 lanes.
__device__ __forceinline__ float max4(float a) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  a = fmaxf(a, dpp(a, std::integral_constant<int, 0xB1>{}));      // quad_perm [1, 0, 3, 2]
  return fmaxf(a, dpp(a, std::integral_constant<int, 0x4E>{}));   // quad_perm [2, 3, 0, 1]
}

// ---------------------------------------------------------------------------
// The rule: e = floor(log2(max |x|)) - 2, limited to [-127, 125] (6 * 2^125 is finite in bf16 and
// fp32); scale code e + 127 in 0 .. 252; element = x / 2^e to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, half to
// even, 6 from 5 up.  NaN elements count as 0, infinite ones become 6 * 2^125 of their sign.
// The conversion rounds and saturates so by itself (measured on every boundary and 200,000 random
// floats: only NaN differs, which it turns into 6), and uses its scale operand's exponent field only.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t kv4_scale_code(float amax) {
  const int s = (int)(__float_as_uint(amax) >> 23) - 2;          // (a subnormal or zero amax: below 0)
  return (uint32_t)min(max(s, 0), 252);
}

// 8 values of a block -> their codes (value i in bits 4i .. 4i + 3).
__device__ __forceinline__ uint32_t kv4_encode8(const float (&x)[8], uint32_t sc) {
  const float s = __uint_as_float((sc << 23) | 0x400000u);       // (code 0: a subnormal acts as 2^-127)
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
}

template <bool F32>
__device__ __forceinline__ void kv4_load8(float (&x)[8], const void* base, int64_t off) {
  if constexpr (F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const v4i w = *reinterpret_cast<const v4i*>(static_cast<const uint16_t*>(base) + off);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float((uint32_t)w[i] << 16);
      x[2 * i + 1] = __uint_as_float((uint32_t)w[i] & 0xffff0000u);
    }
  }
}

// One thread per 8 elements of K and the same 8 of V, 4 lanes to a block; consecutive threads walk a
// token, then the tokens of a head, so a wave's codes are contiguous.
template <bool F32>
__device__ __forceinline__ void kv4_append_impl(const Kv4CopyArgs& a) {
  const uint32_t cpr = (uint32_t)a.D / 8, u = blockIdx.x * 256 + threadIdx.x;
  const uint32_t c = u % cpr, row = u / cpr;
  const uint32_t t = row % (uint32_t)a.n, bh = row / (uint32_t)a.n;
  if (bh >= (uint32_t)a.B * a.H) return;                         // whole 4-lane groups leave together
  const uint32_t b = bh / (uint32_t)a.H, h = bh % (uint32_t)a.H;
  const int64_t at = (int64_t)(a.pos ? a.pos[b] : a.pos0) + t;
  if ((a.counts && (int)t >= a.counts[b]) || at < 0 || at >= a.L) return;
  float xk[8], xv[8];
  kv4_load8<F32>(xk, a.kx, b * a.k_b + h * a.k_h + t * a.k_t + 8 * c);
  kv4_load8<F32>(xv, a.vx, b * a.v_b + h * a.v_h + t * a.v_t + 8 * c);
  auto put = [&](float (&x)[8], uint8_t* codes, uint8_t* scales) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[i] = x[i] == x[i] ? x[i] : 0.0f;
      m = fmaxf(m, fabsf(x[i]));
    }
    const uint32_t sc = kv4_scale_code(max4(m));
    *reinterpret_cast<uint32_t*>(codes + ((int64_t)bh * a.L + at) * (a.D / 2) + 4 * c) = kv4_encode8(x, sc);
    if ((c & 3) == 0) scales[(int64_t)bh * a.L * (a.D / 32) + kv4_scale_at((int)at, (int)(c >> 2), a.D / 32)] = (uint8_t)sc;
  };
  put(xk, a.k, a.ks);
  put(xv, a.v, a.vs);
}

extern "C" __global__ void __launch_bounds__(256) mxfa_kv4_append_f32(Kv4CopyArgs a) { kv4_append_impl<true>(a); }
extern "C" __global__ void __launch_bounds__(256) mxfa_kv4_append_bf16(Kv4CopyArgs a) { kv4_append_impl<false>(a); }

// The inverse: one thread per 8 elements of K and of V.  Rows outside the cache are 0.
template <bool F32>
__device__ __forceinline__ void kv4_read_impl(const Kv4CopyArgs& a) {
  const uint32_t cpr = (uint32_t)a.D / 8, u = blockIdx.x * 256 + threadIdx.x;
  const uint32_t c = u % cpr, row = u / cpr;
  const uint32_t t = row % (uint32_t)a.n, bh = row / (uint32_t)a.n;
  if (bh >= (uint32_t)a.B * a.H) return;
  const uint32_t b = bh / (uint32_t)a.H, h = bh % (uint32_t)a.H;
  const int64_t at = (int64_t)(a.pos ? a.pos[b] : a.pos0) + t;
  const bool in = at >= 0 && at < a.L;
  uint32_t wk = 0, wv = 0, sk = 0, sv = 0;
  if (in) {
    const int64_t ca = ((int64_t)bh * a.L + at) * (a.D / 2) + 4 * c;
    const int64_t sa = (int64_t)bh * a.L * (a.D / 32) + kv4_scale_at((int)at, (int)(c >> 2), a.D / 32);
    wk = *reinterpret_cast<const uint32_t*>(a.k + ca);
    wv = *reinterpret_cast<const uint32_t*>(a.v + ca);
    sk = a.ks[sa];
    sv = a.vs[sa];
  }
  auto put = [&](uint32_t w, uint32_t sc, void* out, int64_t off) {
    const float s = e8m0_as_float(sc);
    if constexpr (F32) {
      const v2f x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
      const v2f x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + off);
      p[0] = make_float4(x0[0], x0[1], x1[0], x1[1]);
      p[1] = make_float4(x2[0], x2[1], x3[0], x3[1]);
    } else {
      v4i x;
      x[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
      x[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
      x[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
      x[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
      *reinterpret_cast<v4i*>(static_cast<uint16_t*>(out) + off) = x;
    }
  };
  put(wk, sk, a.kx, b * a.k_b + h * a.k_h + t * a.k_t + 8 * c);
  put(wv, sv, a.vx, b * a.v_b + h * a.v_h + t * a.v_t + 8 * c);
}

extern "C" __global__ void __launch_bounds__(256) mxfa_kv4_read_f32(Kv4CopyArgs a) { kv4_read_impl<true>(a); }
extern "C" __global__ void __launch_bounds__(256) mxfa_kv4_read_bf16(Kv4CopyArgs a) { kv4_read_impl<false>(a); }

// ---------------------------------------------------------------------------
// Attention, streaming form.  The query rows of a KV head (row r: query r / group of head r %
// group) are taken 16 at a time as the columns of S^T = K Q^T and O^T += V^T P^T on the 16x16x32 bf16
// MFMA; K and V are widened to bf16 (exact) in registers, never through LDS.  Lane (n, g) = (lane %
// 16, lane / 16):
//   A operand: row n, k = 8 g + e (e < 8); B: column n, k likewise; C: column n, rows 4 g + i (i < 4).
// Row 4 g + i of a 16-key score tile t of a 32-key group is key 16 t + 4 i + g, so a lane's 8 scores of a
// group are the keys = g (mod 4); with k = 8 g + 4 t + i of the PV product the same keys, P goes from the
// score's registers into its operand without a move between lanes, and the V rows that one load
// instruction reads (fixed t, i) are four consecutive keys: whole lines.  The contraction over d may
// take any order: lane (n, g) reads its part of K row n as one piece of at most 16 bytes.
//
// The softmax keeps a reference exponent `mc` for each column instead of the running maximum: it is
// raised (with O and l rescaled) only when a score exceeds it by more than kSlack binades, so P stays
// below 2^kSlack and a block's maximum crosses lanes only then.
// ---------------------------------------------------------------------------
constexpr float kSlack = 4.0f;
constexpr int KV4_NW = 4;            // waves of a workgroup, each its own key blocks
constexpr int KV4_BK = 64;           // keys of a block

__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t cvt_fp4_bf16(uint32_t w, float s, int byte) {
  switch (byte) {                    // (the selector is an immediate; folds away)
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
  }
}

// Byte i of w as the exponent field of a conversion's scale operand, which uses nothing else of it (sign
// and mantissa hold other bits of w).
__device__ __forceinline__ float scale_byte(uint32_t w, int i) {
  return __uint_as_float(i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  v2bf t;
  t[0] = (__bf16)a;
  t[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, t);
}

// Maximum over the four lanes of a column (n, n + 16, n + 32, n + 48).
__device__ __forceinline__ float col_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return pair_max(x);
}

// Range of a row tile's keys: [lo, hi] of one query position of sequence length `len`.
__device__ __forceinline__ void kv4_limits(const Kv4AttnArgs& a, int len, int pos0, int i, int& lo, int& hi) {
  const int qpos = pos0 + i;
  hi = a.causal ? min(len - 1, qpos) : len - 1;
  lo = a.window > 0 ? max(0, qpos - a.window + 1) : 0;
}

// PT: bf16 terms of P in the PV product.
template <int D, bool SOFTCAP, int PT>
__device__ __forceinline__ void kv4_attn_impl(const Kv4AttnArgs& a) {
  constexpr int NW = KV4_NW, BK = KV4_BK;
  constexpr int KD = D / 32;             // K dwords of a lane and row: MFMAs of the score
  constexpr int VB = D / 32;             // V bytes of a lane and row: 2 VB elements of d
  constexpr int NB = D / 32;             // MX blocks of a row
  constexpr int ND = D / 16;             // d tiles of O^T
  constexpr int OP = D + 4;              // row pitch of the merge tile (floats)
  __shared__ __attribute__((aligned(16))) float so[NW][16][OP];
  __shared__ float sml[NW][16][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int part = blockIdx.x % a.n_parts, item = blockIdx.x / a.n_parts;
  const int rt = item % a.n_rt, bk = item / a.n_rt;
  const int b = bk / a.Hkv, kvh = bk % a.Hkv;
  const int len = a.kv_len ? min(max(a.kv_len[b], 0), a.Sk) : a.Sk;
  const int pos0 = a.kv_len ? len - a.Sq : a.q_pos0;
  const int row0 = rt * 16, row = row0 + n, nrow = min(16, a.rows - row0);
  const bool valid = n < nrow;
  const int qi = (valid ? row : row0) / a.group, hd = kvh * a.group + (valid ? row : row0) % a.group;

  // this column's keys, and those that every column of the tile sees or any does
  int klo, khi, klo_all, khi_all, klo_any, khi_any;
  kv4_limits(a, len, pos0, qi, klo, khi);
  kv4_limits(a, len, pos0, row0 / a.group, klo_any, khi_all);
  kv4_limits(a, len, pos0, (row0 + nrow - 1) / a.group, klo_all, khi_any);

  // Q: column n, k of MFMA kk: d = qd(kk) + e
  v4i q[KD];
  const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_b + hd * a.q_h + qi * a.q_t;
#pragma unroll
  for (int kk = 0; kk < KD; kk++) {
    const int d = D == 256 ? (kk >> 2) * 128 + g * 32 + 8 * (kk & 3) : g * (D / 4) + 8 * kk;
    q[kk] = valid ? *reinterpret_cast<const v4i*>(qp + d) : (v4i){0, 0, 0, 0};
  }

  const int64_t bytes = (int64_t)a.L * (D / 2), sbytes = (int64_t)a.L * NB;
  const __amdgpu_buffer_rsrc_t rk = buf_rsrc(a.k, bk * bytes, bytes), rv = buf_rsrc(a.v, bk * bytes, bytes);
  const __amdgpu_buffer_rsrc_t rks = buf_rsrc(a.ks, bk * sbytes, sbytes), rvs = buf_rsrc(a.vs, bk * sbytes, sbytes);

  uint32_t kr[4][KD], ksr[2][D == 256 ? 2 : 1];
  uint32_t vr[2][8][VB > 4 ? 2 : 1];
  v2i vsr[2];
  // A disabled load gets an offset past every resource: it reads nothing and returns 0.
  auto load_k = [&](int key0, bool on) {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int key = key0 + 32 * (t >> 1) + 16 * (t & 1) + 4 * (n & 3) + (n >> 2);
      const uint32_t o = on ? (uint32_t)(key * (D / 2)) : 0x80000000u;
      if constexpr (D == 64) {
        const v2i w = __builtin_amdgcn_raw_buffer_load_b64(rk, o + 8 * g, 0, 0);
        kr[t][0] = w[0]; kr[t][1] = w[1];
      } else {
#pragma unroll
        for (int c = 0; c < KD / 4; c++) {
          const v4i w = __builtin_amdgcn_raw_buffer_load_b128(rk, o + 64 * c + 16 * g, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; i++) kr[t][4 * c + i] = w[i];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint32_t o = on ? (uint32_t)((key0 / 32 + u) * (32 * NB) + 2 * (n & 3)) : 0x80000000u;
#pragma unroll
      for (int c = 0; c < (D == 256 ? 2 : 1); c++)
        ksr[u][c] = __builtin_amdgcn_raw_buffer_load_b16(rks, o + 8 * ((n >> 2) * NB + (D == 64 ? g >> 1 : 4 * c + g)), 0, 0);
    }
  };
  auto load_v = [&](int key0, bool on) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int key = key0 + 32 * u + 16 * (e >> 2) + 4 * (e & 3) + g;
        const uint32_t o = on ? (uint32_t)(key * (D / 2) + n * VB) : 0x80000000u;
        if constexpr (VB == 2)
          vr[u][e][0] = __builtin_amdgcn_raw_buffer_load_b16(rv, o, 0, 0);
        else if constexpr (VB == 4)
          vr[u][e][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, 0, 0);
        else {
          const v2i w = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, 0);
          vr[u][e][0] = w[0]; vr[u][e][1] = w[1];
        }
      }
      const uint32_t o = on ? (uint32_t)((key0 / 32 + u) * (32 * NB) + 8 * (g * NB + n * NB / 16)) : 0x80000000u;
      vsr[u] = __builtin_amdgcn_raw_buffer_load_b64(rvs, o, 0, 0);
    }
  };

  v4f o[ND];
#pragma unroll
  for (int j = 0; j < ND; j++) o[j] = (v4f){0, 0, 0, 0};
  float mc = -INFINITY, l = 0.0f;
  const float c = SOFTCAP ? 1.0f : a.c_log2;

  // blocks of this wave: first, first + step, ... while their first key is at most khi_any
  const int step = a.n_parts * NW * BK;
  const int kfirst = (klo_any / BK + part * NW + wave) * BK;
  load_k(kfirst, kfirst <= khi_any);
  load_v(kfirst, kfirst <= khi_any);
  for (int key0 = kfirst; key0 <= khi_any; key0 += step) {
    const bool more = key0 + step <= khi_any;
    // ---- S^T
    v4f s[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      s[t] = (v4f){0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KD; kk++) {
        const float sc = scale_byte(ksr[t >> 1][D == 256 ? kk >> 2 : 0], t & 1);
        v4i ka;
#pragma unroll
        for (int i = 0; i < 4; i++) ka[i] = (int)cvt_fp4_bf16(kr[t][kk], sc, i);
        s[t] = mfma16(ka, q[kk], s[t]);
      }
    }
    load_k(key0 + step, more);
    if (SOFTCAP) {
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float u = s[t][i] * a.sc_u;
          const float e = __builtin_amdgcn_exp2f(-2.0f * LOG2E_F * fabsf(u));
          const float th = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
          s[t][i] = a.cap_log2 * (u < 0.0f ? -th : th);
        }
    }
    if (key0 < klo_all || key0 + BK - 1 > khi_all) {
      // masked scores to -inf; the scales of V rows that no query of the tile may see (what lies there may
      // be anything) to 2^-127, so that their product with P = 0 is 0
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int key = key0 + 16 * t + 4 * i + g;
          s[t][i] = key >= klo && key <= khi ? s[t][i] : -INFINITY;
        }
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int by = 2 * (e & 3) + (e >> 2);
          const int key = key0 + 32 * u + 16 * (e >> 2) + 4 * (e & 3) + g;
          if (key < klo_any || key > khi_any) vsr[u][by >> 2] &= ~(0xff << (8 * (by & 3)));
        }
    }
    // ---- reference exponent
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][i]);
    if (__any(__builtin_fmaf(mx, c, -mc) > kSlack)) {
      // (by the column's own maximum: a row's result does not depend on its neighbours in the tile)
      const float top = col_max(mx);
      const bool up = __builtin_fmaf(top, c, -mc) > kSlack;
      const float corr = up ? __builtin_amdgcn_exp2f(mc - top * c) : 1.0f;
      mc = up ? top * c : mc;
      l *= corr;
#pragma unroll
      for (int j = 0; j < ND; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[j][i] *= corr;
    }
    const float mcn = mc == -INFINITY ? 0.0f : -mc;
    // ---- P: its terms as B operands of the two 32-key products
    v4i p[2][PT];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const int t = 2 * u + (x >> 1), i = 2 * (x & 1);
        float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, mcn));
        float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i + 1], c, mcn));
        if constexpr (PT > 1) l += p0 + p1;
#pragma unroll
        for (int y = 0; y < PT; y++) {
          const uint32_t w = pack_bf16(p0, p1);
          p[u][y][x] = (int)w;
          const float r0 = __uint_as_float(w << 16), r1 = __uint_as_float(w & 0xffff0000u);
          if constexpr (PT == 1) l += r0 + r1;
          p0 -= r0;
          p1 -= r1;
        }
      }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float sc[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int by = 2 * (e & 3) + (e >> 2);
        sc[e] = scale_byte((uint32_t)vsr[u][by >> 2], by & 3);
      }
#pragma unroll
      for (int by = 0; by < VB; by++) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = cvt_fp4_bf16(vr[u][e][by >> 2], sc[e], by & 3);
        v4i v0, v1;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          v0[x] = (int)__builtin_amdgcn_perm(w[2 * x + 1], w[2 * x], 0x05040100u);
          v1[x] = (int)__builtin_amdgcn_perm(w[2 * x + 1], w[2 * x], 0x07060302u);
        }
#pragma unroll
        for (int y = 0; y < PT; y++) {
          o[2 * by] = mfma16(v0, p[u][y], o[2 * by]);
          o[2 * by + 1] = mfma16(v1, p[u][y], o[2 * by + 1]);
        }
      }
    }
    load_v(key0 + step, more);
  }

  // ---- merge the waves: d = (4 g + i) ND + j of column n
  l += __shfl_xor(l, 16);
  l = pair_sum(l);
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < ND; j += 4)
      *reinterpret_cast<float4*>(&so[wave][n][(4 * g + i) * ND + j]) = make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]);
  if (g == 0) {
    sml[wave][n][0] = mc;
    sml[wave][n][1] = l;
  }
  __syncthreads();
  // thread (col, x) = (tid / 16, tid % 16): 4 consecutive d at 4 x, 4 x + 64, ...
  const int col = tid >> 4, d0 = 4 * (tid & 15);
  if (col >= nrow) return;
  float M = -INFINITY, L = 0.0f, wt[NW];
#pragma unroll
  for (int w = 0; w < NW; w++) M = fmaxf(M, sml[w][col][0]);
#pragma unroll
  for (int w = 0; w < NW; w++) {
    wt[w] = __builtin_amdgcn_exp2f(sml[w][col][0] - (M == -INFINITY ? 0.0f : M));
    L += sml[w][col][1] * wt[w];
  }
  const int r = row0 + col;
  const int64_t pr = ((int64_t)bk * a.rows + r) * a.n_parts + part;
  const int64_t oo = b * a.o_b + (kvh * a.group + r % a.group) * a.o_h + r / a.group * a.o_t;
#pragma unroll
  for (int d = d0; d < D; d += 64) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float4 x = *reinterpret_cast<const float4*>(&so[w][col][d]);
      acc.x += x.x * wt[w]; acc.y += x.y * wt[w]; acc.z += x.z * wt[w]; acc.w += x.w * wt[w];
    }
    if (a.n_parts > 1) {
      *reinterpret_cast<float4*>(a.part_o + pr * D + d) = acc;
    } else {
      const float inv = L != 0.0f ? 1.0f / L : 0.0f;             // no visible key: 0
      acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
      if (a.o_bf16)
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + oo + d) = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
      else
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.o) + oo + d) = acc;
    }
  }
  if (a.n_parts > 1 && d0 == 0) {
    a.part_ml[2 * pr] = M;
    a.part_ml[2 * pr + 1] = L;
  }
}

#define MXFA_KV4_ATTN(D, SC, PT, NAME) \
  extern "C" __global__ void __launch_bounds__(256, 2) NAME(Kv4AttnArgs a) { kv4_attn_impl<D, SC, PT>(a); }
#define MXFA_KV4_ATTN_ALL(D)                                            \
  MXFA_KV4_ATTN(D, false, 2, mxfa_kv4_attn_d##D)                        \
  MXFA_KV4_ATTN(D, true, 2, mxfa_kv4_attn_d##D##_softcap)               \
  MXFA_KV4_ATTN(D, false, 3, mxfa_kv4_attn_d##D##_f32)                  \
  MXFA_KV4_ATTN(D, true, 3, mxfa_kv4_attn_d##D##_softcap_f32)
MXFA_KV4_ATTN_ALL(64)
MXFA_KV4_ATTN_ALL(128)
MXFA_KV4_ATTN_ALL(256)

// O = sum_p O_p 2^(m_p - M) / sum_p l_p 2^(m_p - M) of the parts of each row; 0 where nothing was visible.
// One workgroup of D threads per row, D / 4 lanes of 4 d for each of 4 groups that take every fourth part.
extern "C" __global__ void __launch_bounds__(256) mxfa_kv4_combine(Kv4AttnArgs a) {
  __shared__ __attribute__((aligned(16))) float so[3][256];
  __shared__ float sl[3];
  const int D = blockDim.x, lanes = D / 4, grp = threadIdx.x / lanes, x = threadIdx.x % lanes;
  const int bk = blockIdx.x / a.rows, r = blockIdx.x % a.rows;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (int64_t)blockIdx.x * a.n_parts;
  const float* po = a.part_o + (int64_t)blockIdx.x * a.n_parts * D + 4 * x;
  float M = -INFINITY;
  for (int p = 0; p < a.n_parts; p++) M = fmaxf(M, ml[p].x);
  const float m0 = M == -INFINITY ? 0.0f : M;
  float L = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = grp; p < a.n_parts; p += 4) {
    const float w = __builtin_amdgcn_exp2f(ml[p].x - m0);
    L += ml[p].y * w;
    const float4 o = *reinterpret_cast<const float4*>(po + (int64_t)p * D);
    acc.x += o.x * w; acc.y += o.y * w; acc.z += o.z * w; acc.w += o.w * w;
  }
  if (grp) {
    *reinterpret_cast<float4*>(&so[grp - 1][4 * x]) = acc;
    if (x == 0) sl[grp - 1] = L;
  }
  __syncthreads();
  if (grp) return;
  for (int i = 0; i < 3; i++) {
    const float4 o = *reinterpret_cast<const float4*>(&so[i][4 * x]);
    acc.x += o.x; acc.y += o.y; acc.z += o.z; acc.w += o.w;
    L += sl[i];
  }
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
  const int b = bk / a.Hkv, kvh = bk % a.Hkv;
  const int64_t oo = b * a.o_b + (kvh * a.group + r % a.group) * a.o_h + r / a.group * a.o_t + 4 * x;
  if (a.o_bf16)
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + oo) = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
  else
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.o) + oo) = acc;
}
