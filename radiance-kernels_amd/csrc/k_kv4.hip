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
// token, then the tokens of a head, so a wave's codes are contiguous.  Bound by memory: 4 x up to 4,096 tokens of
// 8 heads, D = 128, bf16, 77 MB in 18 us (4.2 TB/s; a copy 5.1); one token of 64 sequences 3.4 us, a launch's time.
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

// The inverse: one thread per 8 elements of K and of V.  Rows outside the cache are 0.  Bound by memory: 8 x 8,192
// tokens of 8 heads, D = 128, to bf16, 340 MB in 62 us (5.5 TB/s).
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
// Attention, streaming form: at most 32 query rows of a KV head (row r: query r / group of head r %
// group), NT tiles of 16 of them as the columns of S^T = K Q^T and O^T += V^T P^T on the 16x16x32 bf16
// MFMA.  K and V are widened to bf16 (exact) in registers, never through LDS.  Lane (n, g) = (lane %
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
//
// Work is dealt in 64-key blocks, an item (sequence, KV head) being as many as its queries see, at least one: a
// workgroup per item, or, where that would leave CUs idle, the blocks of all items shared out over as many
// workgroups as the chip holds, whatever the lengths (kv4_share).  A workgroup's four waves take every fourth block of
// a piece and merge through LDS; a piece that is a whole item is written out, others go to the workspace and
// mxfa_kv4_combine merges them.
//
// What bounds it: memory, for up to 16 rows.  64 x 8,192 tokens, 32 heads on 8 of D = 128: 571 MB in 88 us, 6.5 TB/s
// (the same loads with nothing else done take 86).  One sequence of 131,072 tokens: 143 MB in 27 us, of which 3 pass
// before a workgroup's first block arrives and 3 after its last; the merge takes 4.5 more.  24 sequences of up to
// 7,000 tokens, D = 256, window 4,096, softcap, fp32 O: 38 us, the blocks themselves 21 of them at the memory's rate.  With
// two tiles the MFMAs and conversions count: 16 drafts of 5 tokens, 55 MB in 21 us, MFMA busy 22%.
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

// Two floats to bf16, nearest even (a in the low half).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2bf));
}

// Maximum over the four lanes of a column (n, n + 16, n + 32, n + 48).
__device__ __forceinline__ float col_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return pair_max(x);
}

// The keys that query i of a sequence sees: [lo, hi].
struct Kv4Seq {
  int len, pos0;
};
// Keys of sequence b.
__device__ __forceinline__ int kv4_len(const Kv4AttnArgs& a, int b) { return a.kv_len ? min(max(a.kv_len[b], 0), a.Sk) : a.Sk; }
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, int len) { return {len, a.kv_len ? len - a.Sq : a.q_pos0}; }
__device__ __forceinline__ void kv4_limits(const Kv4AttnArgs& a, Kv4Seq s, int i, int& lo, int& hi) {
  hi = a.causal ? min(s.len - 1, s.pos0 + i) : s.len - 1;
  lo = a.window > 0 ? max(0, s.pos0 + i - a.window + 1) : 0;
}

// Items are (sequence, row tile, KV head), the heads fastest; `gt` = sequence * n_rt + row tile.  First and last
// query of a row tile, and the 64-key blocks that its items walk (the first query sees the lowest key, the last
// the highest).
__device__ __forceinline__ void kv4_tile(const Kv4AttnArgs& a, int gt, int& b, int& row0, int& i0, int& i1) {
  b = a.n_rt == 1 ? gt : gt / a.n_rt;
  row0 = a.n_rt == 1 ? 0 : (gt - b * a.n_rt) * a.tile_rows;
  i0 = a.n_rt == 1 ? 0 : row0 / a.group;
  i1 = a.n_rt == 1 ? a.Sq - 1 : (min(row0 + a.tile_rows, a.rows) - 1) / a.group;
}
__device__ __forceinline__ int kv4_blocks(const Kv4AttnArgs& a, int gt, int len) {
  int b, row0, i0, i1, lo, hi, t;
  kv4_tile(a, gt, b, row0, i0, i1);
  const Kv4Seq s = kv4_seq(a, len);
  kv4_limits(a, s, i0, lo, t);
  kv4_limits(a, s, i1, t, hi);
  return hi >= lo ? hi / KV4_BK - lo / KV4_BK + 1 : 1;
}
__device__ __forceinline__ int kv4_tile_len(const Kv4AttnArgs& a, int gt) { return kv4_len(a, a.n_rt == 1 ? gt : gt / a.n_rt); }
// What an item takes up in the line: its blocks and, short ones, room for the time that a piece costs by itself
// (Q, the first loads, the merge: some 8 blocks' worth), so that a share does not hold many of them.
__device__ __forceinline__ int kv4_room(int nblk) { return nblk < 32 ? nblk + 8 : nblk; }

// Inclusive prefix sum over a wave, by DPP (shifts inside rows of 16, then the row totals broadcast on).
__device__ __forceinline__ int wave_prefix(int x) {
  auto add = [&](auto ctrl, auto rows) { x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false); };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});   // row_shr:1
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});   // row_shr:2
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});   // row_shr:4
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});   // row_shr:8
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});   // row_bcast:15 to rows 1 and 3
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});   // row_bcast:31 to rows 2 and 3
  return x;
}
// How the blocks are dealt.  With few items (a.cut: at most half as many as workgroups), each is cut into pieces of equal
// size, a multiple of the waves, and every piece is a workgroup of its own: `share` is the smallest size (to a
// sixteenth) with which there are workgroups for all pieces.  With more items the line of all of them is cut into
// equal shares, each a workgroup that walks the pieces in it.  (Ragged batches of up to 4,096 tokens, 8 KV heads of D = 128,
// us, line and cut: 192 items 22.3, 19.1; 256 items 23.8, 22.4; 384 items 29.0, 30.8.)
__device__ __forceinline__ uint32_t kv4_pieces(uint32_t nblk, uint32_t share) { return (nblk + share - 1) / share; }
__device__ __forceinline__ uint32_t kv4_up(uint32_t n) { return (n + KV4_NW - 1) / KV4_NW * KV4_NW; }
// nblk0: kv4_blocks of tile `lane` (0 past the last).
__device__ __forceinline__ uint32_t kv4_share(const Kv4AttnArgs& a, int lane, uint32_t nblk0) {
  const int groups = a.B * a.n_rt;
  auto sum = [&](auto f) {
    uint32_t n = nblk0 ? f(nblk0) : 0;
    for (int gt = 64 + lane; gt < groups; gt += 64) n += f(kv4_blocks(a, gt, kv4_tile_len(a, gt)));
    return __builtin_amdgcn_readlane(wave_prefix(n), 63) * (uint32_t)a.Hkv;
  };
  const uint32_t total = sum([&](uint32_t n) { return a.cut ? n : kv4_room(n); });
  uint32_t s = max(kv4_up((total + a.n_wg - 1) >> a.wg_log2), (uint32_t)a.min_share);
  if (a.cut) {
    const uint32_t step = kv4_up(s >> 4);
    while (sum([&](uint32_t n) { return kv4_pieces(n, s); }) > (uint32_t)a.n_wg) s += step;
  }
  return s;
}

// This workgroup's part of the line: `left` places from j0 of item (row tile gt, KV head kvh) on; an item's later pieces
// hold `share`; len: its keys.  False: none.
struct Kv4Part {
  int gt, kvh, j0, left, share, len;
};
__device__ __forceinline__ bool kv4_my_part(const Kv4AttnArgs& a, int lane, Kv4Part& w) {
  if (!a.n_wg) {                           // one workgroup per item, the tiles that see most keys first
    w.gt = a.B * a.n_rt - 1 - blockIdx.x / a.Hkv;
    w.kvh = blockIdx.x % a.Hkv;
    w.j0 = 0;
    w.len = __builtin_amdgcn_readfirstlane(kv4_tile_len(a, w.gt));
    w.left = w.share = kv4_room(kv4_blocks(a, w.gt, w.len));
    return true;
  }
  const int groups = a.B * a.n_rt;
  int len = kv4_tile_len(a, min(lane, groups - 1));
  uint32_t nblk = lane < groups ? kv4_blocks(a, lane, len) : 0;
  const uint32_t share = kv4_share(a, lane, nblk), u0 = a.cut ? blockIdx.x : blockIdx.x * share;
  uint32_t at = 0;                         // places (cut: pieces) before tile g0
  for (int g0 = 0; g0 < groups; g0 += 64) {
    if (g0) {
      len = kv4_tile_len(a, min(g0 + lane, groups - 1));
      nblk = g0 + lane < groups ? kv4_blocks(a, g0 + lane, len) : 0;
    }
    const uint32_t each = !nblk ? 0 : a.cut ? kv4_pieces(nblk, share) : kv4_room(nblk), mine = each * a.Hkv;
    const uint32_t sum = wave_prefix(mine);
    const uint64_t past = __ballot(at + sum > u0);
    if (past) {
      const int l = __builtin_ctzll(past);
      const uint32_t n = __builtin_amdgcn_readlane(nblk, l), per = __builtin_amdgcn_readlane(each, l);
      const uint32_t in = u0 - (at + __builtin_amdgcn_readlane(sum, l) - per * a.Hkv);
      w.gt = g0 + l;
      w.len = __builtin_amdgcn_readlane(len, l);
      w.kvh = in / per;
      w.j0 = in - w.kvh * per;
      w.left = w.share = share;            // (the walk ends at the last tile)
      if (a.cut) {
        const uint32_t size = kv4_up((n + per - 1) / per);
        w.j0 *= size;
        w.share = size;
        w.left = min((int)size, (int)n - w.j0);
        return w.left > 0;
      }
      return true;
    }
    at += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}
// The first piece of an item (nj of its nblk blocks) leaves in the workspace where the item's pieces lie: its own slot
// and their number.  The second lies in slot `a.cut ? w + 1 : 2 (w + 1)` for workgroup w.
__device__ __forceinline__ void kv4_note_item(const Kv4AttnArgs& a, const Kv4Part& w, int nblk, int nj, int slot) {
  if (a.n_wg && w.j0 == 0 && threadIdx.x == 0)
    reinterpret_cast<int2*>(a.pieces)[w.gt * a.Hkv + w.kvh] = make_int2(slot, 1 + (uint32_t)(nblk - nj + w.share - 1) / (uint32_t)w.share);
}

// 4 values of O (query i, head hd) from d on.
__device__ __forceinline__ void kv4_store4(const Kv4AttnArgs& a, int b, int hd, int i, int d, float4 x) {
  const int64_t o = b * a.o_b + hd * a.o_h + i * a.o_t + d;
  if (a.o_bf16)
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + o) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
  else
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.o) + o) = x;
}

// PT: bf16 terms of P in the PV product.
template <int D, int NT, bool SOFTCAP, int PT>
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

  Kv4Part w;
  if (!kv4_my_part(a, lane, w)) return;
  const bool young = (int)blockIdx.x >= 256;   // (the first 256 workgroups take a CU each)
  bool first = true;

  while (true) {
    const int nblk = kv4_blocks(a, w.gt, w.len), b = w.gt, kvh = w.kvh, j0 = w.j0;       // (one row tile)
    const int take = min(kv4_room(nblk) - j0, w.left), nj = min(nblk - j0, take);
    if (nj > 0) {
    const int slot = a.cut ? blockIdx.x : 2 * blockIdx.x + (first ? 0 : 1);
    const int bk = b * a.Hkv + kvh;
    const Kv4Seq seq = kv4_seq(a, w.len);
    // each column's keys, and those that every column sees or any does
    int klo[NT], khi[NT], klo_all, khi_all, klo_any, khi_any;
    kv4_limits(a, seq, 0, klo_any, khi_all);
    kv4_limits(a, seq, a.Sq - 1, klo_all, khi_any);
    // Q: column n, k of MFMA kk: d = qd(kk) + e
    v4i q[NT][KD];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int row = 16 * t + n;
      const bool valid = row < a.rows;
      const int qi = valid ? row * a.group_inv >> 16 : 0, hd = kvh * a.group + (valid ? row - qi * a.group : 0);
      kv4_limits(a, seq, qi, klo[t], khi[t]);
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_b + hd * a.q_h + qi * a.q_t;
#pragma unroll
      for (int kk = 0; kk < KD; kk++) {
        const int d = D == 256 ? (kk >> 2) * 128 + g * 32 + 8 * (kk & 3) : g * (D / 4) + 8 * kk;
        q[t][kk] = valid ? *reinterpret_cast<const v4i*>(qp + d) : (v4i){0, 0, 0, 0};
      }
    }

    const int64_t bytes = (int64_t)a.L * (D / 2), sbytes = (int64_t)a.L * NB;
    const __amdgpu_buffer_rsrc_t rk = buf_rsrc(a.k, bk * bytes, bytes), rv = buf_rsrc(a.v, bk * bytes, bytes);
    const __amdgpu_buffer_rsrc_t rks = buf_rsrc(a.ks, bk * sbytes, sbytes), rvs = buf_rsrc(a.vs, bk * sbytes, sbytes);

    // Codes are read once, whole lines per instruction: non-temporal loads (64 x 8,192 tokens of D = 128:
    // 96 us, 104 with the default policy).
    constexpr int kNT = 2;
    uint32_t kr[4][KD], ksr[2][D == 256 ? 2 : 1];
    uint32_t vr[2][8][VB > 4 ? 2 : 1];
    v2i vsr[2];
    // (Loads from key L on lie past the resources: they read nothing and return 0.)
    const uint32_t klane = (4 * (n & 3) + (n >> 2)) * (D / 2) + (D == 64 ? 8 : 16) * g, vlane = g * (D / 2) + n * VB;
    const uint32_t kslane = 2 * (n & 3) + 8 * ((n >> 2) * NB + (D == 64 ? g >> 1 : g)), vslane = 8 * (g * NB + n * NB / 16);
    auto load_k = [&](int key0) {
      const uint32_t base = klane + (uint32_t)key0 * (D / 2), sbase = kslane + (uint32_t)key0 * NB;
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const uint32_t o = base + 16 * t * (D / 2);
        if constexpr (D == 64) {
          const v2i w = __builtin_amdgcn_raw_buffer_load_b64(rk, o, 0, kNT);
          kr[t][0] = w[0]; kr[t][1] = w[1];
        } else {
#pragma unroll
          for (int c = 0; c < KD / 4; c++) {
            const v4i w = __builtin_amdgcn_raw_buffer_load_b128(rk, o + 64 * c, 0, kNT);
#pragma unroll
            for (int i = 0; i < 4; i++) kr[t][4 * c + i] = w[i];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int c = 0; c < (D == 256 ? 2 : 1); c++)
          ksr[u][c] = __builtin_amdgcn_raw_buffer_load_b16(rks, sbase + 32 * NB * u + 32 * c, 0, 0);
    };
    auto load_v = [&](int key0) {
      const uint32_t base = vlane + (uint32_t)key0 * (D / 2), sbase = vslane + (uint32_t)key0 * NB;
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint32_t o = base + (32 * u + 16 * (e >> 2) + 4 * (e & 3)) * (D / 2);
          if constexpr (VB == 2)
            vr[u][e][0] = __builtin_amdgcn_raw_buffer_load_b16(rv, o, 0, kNT);
          else if constexpr (VB == 4)
            vr[u][e][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, 0, kNT);
          else {
            const v2i w = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, kNT);
            vr[u][e][0] = w[0]; vr[u][e][1] = w[1];
          }
        }
        vsr[u] = __builtin_amdgcn_raw_buffer_load_b64(rvs, sbase + 32 * NB * u, 0, 0);
      }
    };

    v4f o[NT][ND];
    float mc[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int j = 0; j < ND; j++) o[t][j] = (v4f){0, 0, 0, 0};
      mc[t] = -INFINITY;
      l[t] = 0.0f;
    }
    const float c = SOFTCAP ? 1.0f : a.c_log2;

    // this wave's blocks: every NW-th of the piece's nj, from block j0 of the item on
    const int kend = (klo_any / BK + j0 + nj) * BK, kfirst = (klo_any / BK + j0 + wave) * BK;
    // (in this order, as in the loop: the wait for K must not become one for V)
    load_k(kfirst < kend ? kfirst : a.L);
    __builtin_amdgcn_sched_barrier(0);
    load_v(kfirst < kend ? kfirst : a.L);
    __builtin_amdgcn_sched_barrier(0);
    for (int key0 = kfirst; key0 < kend; key0 += NW * BK) {
      // Of two workgroups on a CU the older one's waves are served first and end well before the younger one's, which
      // then has the CU to itself, too few waves to fill it: three blocks of four the younger has priority (64 x 8,192
      // tokens: 94.4 us without, 92.1 so).
      if (young) {
        if (((key0 - kfirst) / (NW * BK) & 3) == 3)
          __builtin_amdgcn_s_setprio(0);
        else
          __builtin_amdgcn_s_setprio(1);
      }
      const int next = key0 + NW * BK < kend ? key0 + NW * BK : a.L;
      const bool masked = key0 < klo_all || key0 + BK - 1 > khi_all;
      // ---- S^T
      v4f s[NT][4];
#pragma unroll
      for (int x = 0; x < 4; x++) {
#pragma unroll
        for (int t = 0; t < NT; t++) s[t][x] = (v4f){0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KD; kk++) {
          const float sc = scale_byte(ksr[x >> 1][D == 256 ? kk >> 2 : 0], x & 1);
          v4i ka;
#pragma unroll
          for (int i = 0; i < 4; i++) ka[i] = (int)cvt_fp4_bf16(kr[x][kk], sc, i);
#pragma unroll
          for (int t = 0; t < NT; t++) s[t][x] = mfma16(ka, q[t][kk], s[t][x]);
        }
      }
      load_k(next);
      v4i p[NT][2][PT];                    // P's terms, B operands of the two 32-key products
#pragma unroll
      for (int t = 0; t < NT; t++) {
        if (SOFTCAP) {
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float u = s[t][x][i] * a.sc_u;
              const float e = __builtin_amdgcn_exp2f(-2.0f * LOG2E_F * fabsf(u));
              const float th = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
              s[t][x][i] = a.cap_log2 * (u < 0.0f ? -th : th);
            }
        }
        if (masked) {
          __asm__ volatile("");            // (keeps the selects behind the branch)
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int key = key0 + 16 * x + 4 * i + g;
              s[t][x][i] = key >= klo[t] && key <= khi[t] ? s[t][x][i] : -INFINITY;
            }
        }
        // ---- reference exponent
        float mx = s[t][0][0];
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][x][i]);
        if (__any(__builtin_fmaf(mx, c, -mc[t]) > kSlack)) {
          // (by the column's own maximum: a row's result does not depend on its neighbours in the tile)
          const float top = col_max(mx);
          const bool up = __builtin_fmaf(top, c, -mc[t]) > kSlack;
          const float corr = up ? __builtin_amdgcn_exp2f(mc[t] - top * c) : 1.0f;
          mc[t] = up ? top * c : mc[t];
          l[t] *= corr;
#pragma unroll
          for (int j = 0; j < ND; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[t][j][i] *= corr;
        }
        const float mcn = mc[t] == -INFINITY ? 0.0f : -mc[t];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int x = 0; x < 4; x++) {
            const int tt = 2 * u + (x >> 1), i = 2 * (x & 1);
            float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][tt][i], c, mcn));
            float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][tt][i + 1], c, mcn));
            l[t] += p0 + p1;
#pragma unroll
            for (int y = 0; y < PT; y++) {
              const uint32_t w = pack_bf16(p0, p1);
              p[t][u][y][x] = (int)w;
              p0 -= __uint_as_float(w << 16);
              p1 -= __uint_as_float(w & 0xffff0000u);
            }
          }
      }
      // ---- O^T += V^T P^T
      uint32_t vw[2][2];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 2; i++) vw[u][i] = (uint32_t)vsr[u][i];
      if (masked) {
        // the scales of V rows that no query may see (what lies there may be anything) to 2^-127, so
        // that their product with P = 0 is 0
        __asm__ volatile("");
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const int by = 2 * (e & 3) + (e >> 2), key = key0 + 32 * u + 16 * (e >> 2) + 4 * (e & 3) + g;
            if (key < klo_any || key > khi_any) vw[u][by >> 2] &= ~(0xffu << (8 * (by & 3)));
          }
      }
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float sc[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int by = 2 * (e & 3) + (e >> 2);
          sc[e] = scale_byte(vw[u][by >> 2], by & 3);
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
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int y = 0; y < PT; y++) {
              o[t][2 * by] = mfma16(v0, p[t][u][y], o[t][2 * by]);
              o[t][2 * by + 1] = mfma16(v1, p[t][u][y], o[t][2 * by + 1]);
            }
        }
      }
      load_v(next);
    }

    // ---- merge the waves, a tile of columns at a time: d = (4 g + i) ND + j of column n
    const bool whole = nj == nblk;
    kv4_note_item(a, w, nblk, nj, slot);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      l[t] += __shfl_xor(l[t], 16);
      l[t] = pair_sum(l[t]);
      __syncthreads();                     // (the tile of the last merge has been read)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < ND; j += 4)
          *reinterpret_cast<float4*>(&so[wave][n][(4 * g + i) * ND + j]) =
              make_float4(o[t][j][i], o[t][j + 1][i], o[t][j + 2][i], o[t][j + 3][i]);
      if (g == 0) {
        sml[wave][n][0] = mc[t];
        sml[wave][n][1] = l[t];
      }
      __syncthreads();
      // thread (col, x) = (tid / 16, tid % 16): 4 consecutive d at 4 x, 4 x + 64, ...
      const int col = tid >> 4, d0 = 4 * (tid & 15), r = 16 * t + col;
      if (r >= a.rows) continue;
      const int qi = r * a.group_inv >> 16;
      float M = -INFINITY, Ls = 0.0f, wt[NW];
#pragma unroll
      for (int w = 0; w < NW; w++) M = fmaxf(M, sml[w][col][0]);
#pragma unroll
      for (int w = 0; w < NW; w++) {
        wt[w] = __builtin_amdgcn_exp2f(sml[w][col][0] - (M == -INFINITY ? 0.0f : M));
        Ls += sml[w][col][1] * wt[w];
      }
      const float inv = !whole ? 1.0f : Ls != 0.0f ? 1.0f / Ls : 0.0f;   // no visible key: 0
#pragma unroll
      for (int d = d0; d < D; d += 64) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
          const float4 x = *reinterpret_cast<const float4*>(&so[w][col][d]);
          acc.x += x.x * wt[w]; acc.y += x.y * wt[w]; acc.z += x.z * wt[w]; acc.w += x.w * wt[w];
        }
        acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
        if (!whole)
          *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * a.tile_rows + r) * D + d) = acc;
        else
          kv4_store4(a, b, kvh * a.group + r - qi * a.group, qi, d, acc);
      }
      if (!whole && d0 == 0) reinterpret_cast<float2*>(a.part_ml)[(int64_t)slot * a.tile_rows + r] = make_float2(M, Ls);
    }
    }
    w.left -= take;
    if (w.left <= 0) return;
    first = false;
    w.j0 = 0;
    if (++w.kvh == a.Hkv) {
      w.kvh = 0;
      if (++w.gt == a.B * a.n_rt) return;
      w.len = __builtin_amdgcn_readfirstlane(kv4_tile_len(a, w.gt));
    }
  }
}

#define MXFA_KV4_ATTN(D, NT, SC, PT, OCC, NAME) \
  extern "C" __global__ void __launch_bounds__(64 * KV4_NW, OCC) NAME(Kv4AttnArgs a) { kv4_attn_impl<D, NT, SC, PT>(a); }
#define MXFA_KV4_ATTN_ALL(D, NT, OCC)                                           \
  MXFA_KV4_ATTN(D, NT, false, 2, OCC, mxfa_kv4_attn_d##D##_t##NT)               \
  MXFA_KV4_ATTN(D, NT, true, 2, OCC, mxfa_kv4_attn_d##D##_t##NT##_softcap)      \
  MXFA_KV4_ATTN(D, NT, false, 3, OCC, mxfa_kv4_attn_d##D##_t##NT##_f32)         \
  MXFA_KV4_ATTN(D, NT, true, 3, OCC, mxfa_kv4_attn_d##D##_t##NT##_softcap_f32)
MXFA_KV4_ATTN_ALL(64, 1, 2)
MXFA_KV4_ATTN_ALL(64, 2, 2)
MXFA_KV4_ATTN_ALL(128, 1, 2)
MXFA_KV4_ATTN_ALL(128, 2, 2)
MXFA_KV4_ATTN_ALL(256, 1, 2)
MXFA_KV4_ATTN_ALL(256, 2, 1)

// ---------------------------------------------------------------------------
// Attention, tiled form: more than 32 query rows of a KV head.  128 rows to a workgroup (32 to each of its four
// waves), 64 keys at a time: the workgroup widens the block's K and V to bf16 (exact) in LDS once, and every
// wave takes S^T = K Q^T and O^T += V^T P^T over its own rows on the 32x32x16 bf16 MFMA, both A operands read
// from LDS.  Lane (n, h) = (lane % 32, lane / 32):
//   A operand: row n, k = 8 h + e (e < 8); B: column n, k likewise; C: column n, rows 8 (i / 4) + 4 h + i % 4.
// V lies transposed, a row of 64 keys for each d, the keys of a 16-key group in the order in which a lane
// holds their scores (8 h + e is key 8 (e / 4) + 4 h + e % 4), so P goes from the score's registers into
// the B operand as it is.  LDS rows are cut into 16-byte units, unit u of K row `key` at u ^ (key & 15) (D = 256:
// the upper 16 units at u ^ ((key ^ 8) & 15); D = 64, rows of 8: u ^ ((key ^ key / 8) & 7)), of V row d, 8 units, at u ^
// ((d ^ d / 8) & 7) of row d ^ (d / 64 & 1): reads and writes of 16 consecutive lanes hit distinct banks.
//
// What bounds it: the MFMAs (33 clocks each) and about as many clocks of 4- and 8-clock VALU work (exponentials,
// conversions), which run beside MFMAs only if an instruction stream has both.  So the scores run a block ahead:
// the MFMAs of block j + 1's scores go between the exponentials of block j, those of block j's PV product
// between the widening of K of block j + 2 and V of block j + 1, whose codes were loaded an iteration before; two
// buffers each, one barrier per block.  1,000 queries of 32 heads on 8 of D = 128 over 16,384 keys: 260 GFLOP in 270 us
// with the merge, 965 TFLOP/s, MFMA busy 48% (widened and multiplied one after the other: 458 us).
// Softmax as in the streaming form, and work dealt alike, items here being row tiles.
// ---------------------------------------------------------------------------
// PT: bf16 terms of P in the PV product.
template <int D, bool SOFTCAP, int PT>
__device__ __forceinline__ void kv4_tiled_impl(const Kv4AttnArgs& a) {
  constexpr int BK = KV4_BK, NB = D / 32, ND = D / 32;
  constexpr int TW = D == 256 ? 2 : 1;     // pieces of K (an MX block) and of V (4 keys x 8 d) that a thread widens
  constexpr int BUF = BK * D * 2;          // bytes of a block's K, and of its V
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * BUF];   // K, K, V, V
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  Kv4Part w;
  if (!kv4_my_part(a, lane, w)) return;
  const bool young = (int)blockIdx.x >= 256;   // (the first 256 workgroups take a CU each)
  bool first = true;

  while (true) {
    const int nblk = kv4_blocks(a, w.gt, w.len), kvh = w.kvh, j0 = w.j0;
    const int take = min(kv4_room(nblk) - j0, w.left), nj = min(nblk - j0, take);
    if (nj > 0) {
      const int slot = a.cut ? blockIdx.x : 2 * blockIdx.x + (first ? 0 : 1);
      int b, row0, i0, i1;
      kv4_tile(a, w.gt, b, row0, i0, i1);
      const int bk = b * a.Hkv + kvh;
      const Kv4Seq seq = kv4_seq(a, w.len);
      int klo_any, khi_any, t0, t1;
      kv4_limits(a, seq, i0, klo_any, t0);
      kv4_limits(a, seq, i1, t1, khi_any);
      // the wave's rows: each column's keys, and those that all of them see (a wave without rows need not mask any)
      const int wrow0 = row0 + wave * 32, wrow1 = min(wrow0 + 32, a.rows) - 1;
      int wlo_all = 0, whi_all = INT32_MAX;
      if (wrow0 < a.rows) {
        kv4_limits(a, seq, wrow0 / a.group, t0, whi_all);
        kv4_limits(a, seq, wrow1 / a.group, wlo_all, t1);
      }
      const int row = wrow0 + n;
      const bool valid = row < a.rows;
      const int qi = valid ? row / a.group : i0, hd = kvh * a.group + (valid ? row % a.group : 0);
      int klo, khi;
      kv4_limits(a, seq, qi, klo, khi);
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_b + hd * a.q_h + qi * a.q_t;
      v4i q[D / 16];
#pragma unroll
      for (int kk = 0; kk < D / 16; kk++) q[kk] = valid ? *reinterpret_cast<const v4i*>(qp + 16 * kk + 8 * h) : (v4i){0, 0, 0, 0};

      const int64_t bytes = (int64_t)a.L * (D / 2), sbytes = (int64_t)a.L * NB;

      // ---- staging.  K: block kbl of key kk0 (D = 64: every piece twice; D = 256: key + 32 too).  V: the 4 keys of half
      // vq % 2 of unit vq / 2, 32 (vq / 8) + 16 (vq / 4 % 2) + 8 (vq % 2) + 4 (vq / 2 % 2) + 0 .. 3, and 8 d from 8 vdc on
      // (D = 64: every piece twice; D = 256: keys + 32 too).
      // (Loads from key L on lie past the resources: they read nothing and return 0.)
      uint32_t kraw[4 * TW], krs[TW], vraw[4 * TW], vrs[4 * TW];
      const int kbl = tid % NB, kk0 = tid / NB & 63, vdc = (tid >> 1) % (D / 8), vq = 2 * (tid / (D / 4) & 7) + (tid & 1);
      const int vk0 = 32 * (vq >> 3) + 16 * ((vq >> 2) & 1) + 8 * (vq & 1) + 4 * ((vq >> 1) & 1);
      const uint32_t klb = kk0 * (D / 2) + 16 * kbl;
      const uint32_t vlb = vk0 * (D / 2) + 4 * vdc;
      // scales: byte x of a group's 8, read as the dword that holds it and turned so that it lies in a float's exponent
      // (a byte load's value would be looked at, to extend it, before it is used, and waited for)
      const uint32_t kx = 2 * ((kk0 >> 2) & 3) + ((kk0 >> 4) & 1), vx = 2 * ((vk0 >> 2) & 3) + ((vk0 >> 4) & 1);
      const uint32_t kls = (kk0 >> 5) * (32 * NB) + ((kk0 & 3) * NB + kbl) * 8 + (kx & 4), kturn = 8 * (kx & 3) + 9 & 31;
      const uint32_t vls = (vk0 >> 5) * (32 * NB) + (vdc >> 2) * 8 + (vx & 4), vturn = 8 * (vx & 3) + 9 & 31;
      auto turned = [](uint32_t w, uint32_t by) { return __uint_as_float(__builtin_amdgcn_alignbit(w, w, by)); };
      // (the block's place goes into the resource, by the scalar unit: a thread's offsets stay the same)
      const uint8_t *kbase = a.k + bk * bytes, *vbase = a.v + bk * bytes, *ksbase = a.ks + bk * sbytes, *vsbase = a.vs + bk * sbytes;
      auto from = [&](const uint8_t* base, int key0, int per) {   // (key0 <= L, L * per < 2^31)
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (uint32_t)(key0 * per)), 0, (a.L - key0) * per, 0x00020000);
      };
      auto load_k = [&](int key0) {
        const __amdgpu_buffer_rsrc_t r = from(kbase, key0, D / 2), rs = from(ksbase, key0, NB);
#pragma unroll
        for (int v = 0; v < TW; v++) {
          const v4i w = __builtin_amdgcn_raw_buffer_load_b128(r, klb + 32 * v * (D / 2), 0, 0);
#pragma unroll
          for (int x = 0; x < 4; x++) kraw[4 * v + x] = (uint32_t)w[x];
          krs[v] = __builtin_amdgcn_raw_buffer_load_b32(rs, kls + 32 * v * NB, 0, 0);
        }
      };
      auto load_v = [&](int key0) {
        const __amdgpu_buffer_rsrc_t r = from(vbase, key0, D / 2), rs = from(vsbase, key0, NB);
#pragma unroll
        for (int i = 0; i < 4 * TW; i++) {
          vraw[i] = __builtin_amdgcn_raw_buffer_load_b32(r, vlb + (32 * (i >> 2) + (i & 3)) * (D / 2), 0, 0);
          vrs[i] = __builtin_amdgcn_raw_buffer_load_b32(rs, vls + (i >> 2) * (32 * NB) + (i & 3) * (8 * NB), 0, 0);
        }
      };
      // V rows of the block at key0 that no query of the tile may see (what lies there may be anything) get scale 2^-127,
      // so that their product with P = 0 is 0
      auto hide_v = [&](int key0) {
        if (key0 < klo_any || key0 + BK - 1 > khi_any) {
          __asm__ volatile("");
#pragma unroll
          for (int i = 0; i < 4 * TW; i++) {
            const int key = key0 + vk0 + 32 * (i >> 2) + (i & 3);
            vrs[i] = key < klo_any || key > khi_any ? 0u : vrs[i];
          }
        }
      };
      // (a unit's place in a row is its number XOR the row's swizzle: rows are aligned to their length)
      uint32_t kst = kk0 * (2 * D) + (kbl >> 2) * 256 +
                     (((D == 64 ? (kk0 ^ (kk0 >> 3)) & 7 : (kk0 ^ 8 * (kbl >> 2)) & 15) ^ (4 * (kbl & 3))) << 4);
      uint32_t vst = 2 * BUF + vdc * 1024 + 128 * ((vdc >> 3) & 1) + (((vq >> 1) ^ (vdc & 7)) << 4) + 8 * (vq & 1);
      auto stage_k = [&](int v, int x) {       // 8 elements of piece v
        v4i w;
#pragma unroll
        for (int y = 0; y < 4; y++) w[y] = (int)cvt_fp4_bf16(kraw[4 * v + x], turned(krs[v], kturn), y);
        *reinterpret_cast<v4i*>(lds + (kst ^ 16 * x) + v * (64 * D)) = w;
      };
      auto stage_v = [&](int v, int by) {      // 2 of the 8 d of piece v
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = cvt_fp4_bf16(vraw[4 * v + e], turned(vrs[4 * v + e], vturn), by);
        const v2i x0 = {(int)__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), (int)__builtin_amdgcn_perm(w[3], w[2], 0x05040100u)};
        const v2i x1 = {(int)__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), (int)__builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
        *reinterpret_cast<v2i*>(lds + (vst ^ (64 * v) ^ (32 * by)) + 256 * by) = x0;
        *reinterpret_cast<v2i*>(lds + (vst ^ (64 * v) ^ (32 * by + 16 + 128)) + 256 * by) = x1;
      };
      auto stage_all = [&](bool with_v) {
#pragma unroll
        for (int u = 0; u < 4 * TW; u++) {
          stage_k(u >> 2, u & 3);
          if (with_v) stage_v(u >> 2, u & 3);
        }
      };
      // (the scales are turned where they are used and not where they are loaded: that would wait for them)
      auto pin = [&] {
#pragma unroll
        for (int i = 0; i < TW; i++) __asm__ volatile("" : "+v"(krs[i]));
#pragma unroll
        for (int i = 0; i < 4 * TW; i++) __asm__ volatile("" : "+v"(vrs[i]));
      };

      // LDS addresses of the A operands: unit h of K row n and of V row n; the other units are an XOR away
      uint32_t kat = n * (2 * D) + ((h ^ (D == 64 ? (n ^ (n >> 3)) & 7 : n & 15)) << 4);
      uint32_t vat = 2 * BUF + n * 128 + ((h ^ ((n ^ (n >> 3)) & 7)) << 4);
      auto kfrag = [&](int f) {                // kk = f / 2, keys 32 (f % 2) + n
        const int kk = f >> 1;
        // (D = 64: key ^ key / 8 of rows 32 on differs from that of row n in bit 2)
        const int i = D == 64 ? (kk ^ 2 * (f & 1)) & 3 : (kk ^ (D == 256 && kk >= 8 ? 4 : 0)) & 7;
        return *reinterpret_cast<const v4i*>(lds + (kat ^ 32 * i) + (kk >> 3) * 256 + (f & 1) * (64 * D));
      };
      auto vfrag = [&](int f) {                // keys of m = f / ND, d = 32 (f % ND) + n
        const int j = f % ND, m = f / ND;
        return *reinterpret_cast<const v4i*>(lds + (vat ^ (32 * (m ^ 2 * (j & 1)) + 128 * ((j >> 1) & 1))) + j * 4096);
      };
      constexpr int NK = D / 8, NV = 4 * ND;   // operands of a block

      v16f o[ND], s[2], t[2];
      float mc = -INFINITY, l = 0.0f;
#pragma unroll
      for (int j = 0; j < ND; j++) o[j] = (v16f){};
      const float c = SOFTCAP ? 1.0f : a.c_log2;
      const int kbeg = (klo_any / BK + j0) * BK, kend = kbeg + nj * BK;
      auto at_or_none = [&](int key0) { return key0 < kend ? min(key0, a.L) : a.L; };   // (a position past the cache: none)

      // ---- before the first block: its K and V and the second one's K widened, its scores
      load_k(at_or_none(kbeg));
      load_v(at_or_none(kbeg));
      pin();
      hide_v(kbeg);
      stage_all(true);
      load_k(at_or_none(kbeg + BK));
      load_v(at_or_none(kbeg + BK));
      __syncthreads();
      s[0] = s[1] = (v16f){};
#pragma unroll
      for (int f = 0; f < NK; f++) s[f & 1] = mfma_bf16(kfrag(f), q[f >> 1], s[f & 1]);
      kst ^= BUF;
      vst ^= BUF;
      kat ^= BUF;
      pin();
      stage_all(false);
      load_k(at_or_none(kbeg + 2 * BK));
      kst ^= BUF;
      __syncthreads();

      auto block = [&](int key0, v16f(&s)[2], v16f(&s2)[2]) {
        if (young) {                           // (as in the streaming form; 290.3 us without, 284.8 so)
          if ((key0 / BK & 3) == 3)
            __builtin_amdgcn_s_setprio(0);
          else
            __builtin_amdgcn_s_setprio(1);
        }
        // s: this block's scores, s2: the next one's.  K of the next block at kat, V of this one at vat; K of the one after next goes to
        // kst, V of the next one to vst.
        if (SOFTCAP) {
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const float u = s[x][i] * a.sc_u;
              const float e = __builtin_amdgcn_exp2f(-2.0f * LOG2E_F * fabsf(u));
              const float th = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
              s[x][i] = a.cap_log2 * (u < 0.0f ? -th : th);
            }
        }
        if (key0 < wlo_all || key0 + BK - 1 > whi_all) {
          __asm__ volatile("");                // (keeps the selects behind the branch)
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int key = key0 + 32 * x + 8 * (i >> 2) + 4 * h + (i & 3);
              s[x][i] = key >= klo && key <= khi ? s[x][i] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[x][i]);
        if (__any(__builtin_fmaf(mx, c, -mc) > kSlack)) {
          const float top = pair_max(mx);
          const bool up = __builtin_fmaf(top, c, -mc) > kSlack;
          const float corr = up ? __builtin_amdgcn_exp2f(mc - top * c) : 1.0f;
          mc = up ? top * c : mc;
          l *= corr;
#pragma unroll
          for (int j = 0; j < ND; j++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[j][i] *= corr;
        }
        const float mcn = mc == -INFINITY ? 0.0f : -mc;
        __asm__ volatile("" : "+v"(kat), "+v"(vat), "+v"(kst), "+v"(vst));   // (the XORs stay here: hoisted, they cost registers)

        // ---- the next block's scores, and between their MFMAs this one's P: its terms as B operands of the four 16-key
        // products.  (Each step is kept together: left to itself the compiler puts the MFMAs first and the rest behind.)
        v4i ka[4], p[4][PT];
#pragma unroll
        for (int f = 0; f < 4; f++) ka[f] = kfrag(f);
        s2[0] = s2[1] = (v16f){};
#pragma unroll
        for (int f = 0; f < NK; f++) {
          s2[f & 1] = mfma_bf16(ka[f & 3], q[f >> 1], s2[f & 1]);
          if (f + 4 < NK) ka[f & 3] = kfrag(f + 4);
#pragma unroll
          for (int g = f * 16 / NK; g < (f + 1) * 16 / NK; g++) {
            const int m = g >> 2, x = g & 3, i = 8 * (m & 1) + 2 * x;
            float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m >> 1][i], c, mcn));
            float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m >> 1][i + 1], c, mcn));
            l += p0;
            l += p1;
#pragma unroll
            for (int y = 0; y < PT; y++) {
              const uint32_t w = pack_bf16(p0, p1);
              p[m][y][x] = (int)w;
              p0 -= __uint_as_float(w << 16);
              p1 -= __uint_as_float(w & 0xffff0000u);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }

        // ---- O^T += V^T P^T, and between its MFMAs the widening
        v4i va[4];
        hide_v(key0 + BK);
        pin();
#pragma unroll
        for (int f = 0; f < 4; f++) va[f] = vfrag(f);
#pragma unroll
        for (int f = 0; f < NV; f++) {
#pragma unroll
          for (int y = 0; y < PT; y++) o[f % ND] = mfma_bf16(va[f & 3], p[f / ND][y], o[f % ND]);
          if (f + 4 < NV) va[f & 3] = vfrag(f + 4);
          constexpr int PER = NV / (8 * TW);   // steps per piece
          if (f % PER == 0) {
            const int u = f / PER, v = u >> 3;
            if (u & 4)
              stage_v(v, u & 3);
            else
              stage_k(v, u & 3);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        load_k(at_or_none(key0 + 3 * BK));
        load_v(at_or_none(key0 + 2 * BK));
        kat ^= BUF;
        vat ^= BUF;
        kst ^= BUF;
        vst ^= BUF;
        __syncthreads();
      };
      for (int key0 = kbeg;; key0 += BK) {
        block(key0, s, t);
        key0 += BK;
        if (key0 >= kend) break;
        block(key0, t, s);
        if (key0 + BK >= kend) break;
      }

      // ---- out: lane (n, h) holds 4 consecutive d of row n in each group of four registers
      const bool whole = nj == nblk;
      kv4_note_item(a, w, nblk, nj, slot);
      const float ls = pair_sum(l);
      if (valid) {
        const float inv = !whole ? 1.0f : ls != 0.0f ? 1.0f / ls : 0.0f;   // no visible key: 0
        const int64_t pr = (int64_t)slot * a.tile_rows + (row - row0);
#pragma unroll
        for (int j = 0; j < ND; j++)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int d = 32 * j + 2 * i + 4 * h;
            const float4 x = make_float4(o[j][i] * inv, o[j][i + 1] * inv, o[j][i + 2] * inv, o[j][i + 3] * inv);
            if (!whole)
              *reinterpret_cast<float4*>(a.part_o + pr * D + d) = x;
            else
              kv4_store4(a, b, hd, qi, d, x);
          }
        if (!whole && h == 0) reinterpret_cast<float2*>(a.part_ml)[pr] = make_float2(mc, ls);
      }
    }
    w.left -= take;
    if (w.left <= 0) return;
    first = false;
    w.j0 = 0;
    if (++w.kvh == a.Hkv) {
      w.kvh = 0;
      if (++w.gt == a.B * a.n_rt) return;
      w.len = __builtin_amdgcn_readfirstlane(kv4_tile_len(a, w.gt));
    }
  }
}

#define MXFA_KV4_TILED(D, SC, PT, OCC, NAME) \
  extern "C" __global__ void __launch_bounds__(256, OCC) NAME(Kv4AttnArgs a) { kv4_tiled_impl<D, SC, PT>(a); }
#define MXFA_KV4_TILED_ALL(D, OCC)                                          \
  MXFA_KV4_TILED(D, false, 1, OCC, mxfa_kv4_tiled_d##D)               \
  MXFA_KV4_TILED(D, true, 1, OCC, mxfa_kv4_tiled_d##D##_softcap)      \
  MXFA_KV4_TILED(D, false, 3, OCC, mxfa_kv4_tiled_d##D##_f32)         \
  MXFA_KV4_TILED(D, true, 3, OCC, mxfa_kv4_tiled_d##D##_softcap_f32)
MXFA_KV4_TILED_ALL(64, 2)
MXFA_KV4_TILED_ALL(128, 2)
MXFA_KV4_TILED_ALL(256, 1)

// The merge of the pieces of an item that several workgroups hold: O = sum O_p 2^(m_p - M) / sum l_p 2^(m_p -
// M); 0 where nothing was visible.  D / 4 lanes hold 4 d each of a row; merge_grp groups of them (a power of two) take
// the row's pieces in turn, the workgroup's other lanes other rows: all lanes for one row after the streaming
// form, where a row may have a piece in every workgroup, one group after the tiled one, whose rows are many
// and have two or three.  blockIdx.y takes a part of the item's rows.  What bounds it is the latency of its loads, one after
// the other: the arguments, the item's note, and the pieces (8 at a time, each group by its own maximum).
extern "C" __global__ void __launch_bounds__(256) mxfa_kv4_combine(Kv4AttnArgs a) {
  __shared__ __attribute__((aligned(16))) float so[256 * 4];
  __shared__ float2 sml[16];
  const int2 item = reinterpret_cast<const int2*>(a.pieces)[blockIdx.x];
  const int slot0 = item.x, np = item.y;
  if (np == 1) return;                     // (written by its workgroup)
  const int lanes = a.D / 4, tid = threadIdx.x, x = tid % lanes, ngrp = a.merge_grp, nrow = 256 / lanes / ngrp;
  const int grp = tid / lanes % ngrp;
  const int gt = blockIdx.x / a.Hkv, kvh = blockIdx.x % a.Hkv;
  int b, row0, i0, i1;
  kv4_tile(a, gt, b, row0, i0, i1);
  const int rows = min(a.tile_rows, a.rows - row0);
  const int slot1 = a.cut ? slot0 : slot0 & ~1, per = a.cut ? 1 : 2;
  constexpr int CH = 8;
  for (int r0 = blockIdx.y * nrow; r0 < rows; r0 += gridDim.y * nrow) {
    const int rr = r0 + tid / lanes / ngrp;   // row in the tile
    const bool have = rr < rows;
    float M = -INFINITY, L = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = grp; p0 < np; p0 += CH * ngrp) {
      float2 v[CH];
      float4 o[CH];
#pragma unroll
      for (int i = 0; i < CH; i++) {
        const int p = p0 + i * ngrp;
        v[i] = make_float2(-INFINITY, 0.f);
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < np) {
          const int64_t at = (int64_t)(p ? slot1 + per * p : slot0) * a.tile_rows + (have ? rr : 0);
          v[i] = reinterpret_cast<const float2*>(a.part_ml)[at];
          o[i] = *reinterpret_cast<const float4*>(a.part_o + at * a.D + 4 * x);
        }
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < CH; i++) top = fmaxf(top, v[i].x);
      const float m0 = top == -INFINITY ? 0.0f : top, old = __builtin_amdgcn_exp2f(M - m0);
      M = top;
      L *= old;
      acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
      for (int i = 0; i < CH; i++) {
        const float w = __builtin_amdgcn_exp2f(v[i].x - m0);
        L += v[i].y * w;
        acc.x += o[i].x * w; acc.y += o[i].y * w; acc.z += o[i].z * w; acc.w += o[i].w * w;
      }
    }
    if (ngrp > 1) {
      __syncthreads();                     // (the last row's sums have been read)
      *reinterpret_cast<float4*>(&so[4 * tid]) = acc;
      if (x == 0) sml[tid / lanes] = make_float2(M, L);
      __syncthreads();
      if (grp == 0) {
        const int g0 = tid / lanes;
        float top = M;
        for (int i = 1; i < ngrp; i++) top = fmaxf(top, sml[g0 + i].x);
        const float m0 = top == -INFINITY ? 0.0f : top;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        L = 0.0f;
        for (int i = 0; i < ngrp; i++) {
          const float4 o = *reinterpret_cast<const float4*>(&so[4 * (tid + i * lanes)]);
          const float w = __builtin_amdgcn_exp2f(sml[g0 + i].x - m0);
          L += sml[g0 + i].y * w;
          acc.x += o.x * w; acc.y += o.y * w; acc.z += o.z * w; acc.w += o.w * w;
        }
      }
    }
    if (grp || !have) continue;
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    const int r = row0 + rr, qi = r / a.group;
    kv4_store4(a, b, kvh * a.group + r - qi * a.group, qi, 4 * x, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
}
