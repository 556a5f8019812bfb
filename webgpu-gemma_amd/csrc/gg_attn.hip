// gg_attn.hip -- attention of new rows over K/V pages.
//
// For a row at position p and the keys j that it sees (j <= p, and with a
// window also j > p - window or j < sinks):
//   s_j = scale q.k_j,  out = sum e^(s_j - m) v_j / sum e^(s_j - m),
// in one pass with a running reference m; O and the sum l are rescaled when a
// step's largest s exceeds m by more than 8 (in log2 units), so weights stay
// below 2^8 and the reference rarely moves. Parts of a long axis are
// joined as O = sum 2^(m_i - M) O_i, l alike.
//
// The heads of a group share a K/V head: (row, head of the group) are packed
// rows, sixteen of them the columns of a matrix instruction. Both products run
// transposed, S^T = K Q^T and O^T = V^T P^T: a lane's results of the first are
// weights of one packed row, and are its operand of the second as they are if
// V's keys are taken in the same order; statistics never cross packed rows.
#include "gg_kv_device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace gg {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;   // log2 units that a score may exceed the reference by

// Parts of a q value and of a weight. bf16 instructions take f32 q in three
// parts of 8 bits, f16 q in two; the weights keep as many bits.
template <int KV, class T>
constexpr int kParts = KV == KV_F16 ? 1 : sizeof(T) == 4 ? 3 : __is_same(T, _Float16) ? 2 : 1;
// f16 weights have 2^7 in them: up to 2^15 with the slack, and down to 2^-31 of
// the reference with any bits.
template <int KV>
constexpr float kShift = KV == KV_F16 ? 7.f : 0.f;

template <int KV>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (KV == KV_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {   // to nearest
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 t;
  t[0] = (__bf16)lo;
  t[1] = (__bf16)hi;
  return __builtin_bit_cast(uint32_t, t);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x2 t;
  t[0] = (_Float16)lo;
  t[1] = (_Float16)hi;
  return __builtin_bit_cast(uint32_t, t);
}
// The upper halves of two words (bf16 towards zero), and the lower ones.
__device__ __forceinline__ uint32_t upper2(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ uint32_t lower2(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }

// Two f32 in NP 16-bit parts (the last one to nearest).
template <int KV, int NP>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&w)[NP]) {
  if constexpr (KV == KV_F16) {
    w[0] = pack_f16(x, y);
  } else {
#pragma unroll
    for (int p = 0; p + 1 < NP; ++p) {
      const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
      w[p] = upper2(xb, yb);
      x -= __uint_as_float(xb & 0xffff0000u);
      y -= __uint_as_float(yb & 0xffff0000u);
    }
    w[NP - 1] = pack_bf16(x, y);
  }
}
// What the first of two 16-bit values, and the second, stand for.
template <int KV>
__device__ __forceinline__ float value_lo(uint32_t w) {
  if constexpr (KV == KV_F16) return f16_lo(w);
  else return __uint_as_float(w << 16);
}
template <int KV>
__device__ __forceinline__ float value_hi(uint32_t w) {
  if constexpr (KV == KV_F16) return f16_hi(w);
  else return __uint_as_float(w & 0xffff0000u);
}

// The keys that some of a tile's rows see, on an axis without the gap between
// the first positions and the window: u < a is position u (below `sink`),
// others are position lo + u - a.
struct Span {
  int lo, a, sink, n;
};
template <int STEP>   // keys that a kernel takes at a time
__device__ __forceinline__ Span kv_span(const KvAttnArgs& g, const KvSeq& sq, int row_first, int row_last) {
  Span s{};
  const int before = sq.len - sq.rows;
  const int hi = min(before + row_last + 1, g.kv.places);
  if (hi <= 0) return s;
  s.lo = g.window > 0 ? max(0, before + row_first - g.window + 1) : 0;
  s.sink = g.window > 0 ? min(min(g.sinks, s.lo), hi) : 0;
  s.a = (s.sink + STEP - 1) / STEP * STEP;
  s.n = s.a + max(0, hi - s.lo);
  return s;
}
__device__ __forceinline__ int kv_splits(const KvAttnArgs& g, const Span& s) { return max(1, (int)g.by_chunk((uint32_t)(s.n + g.chunk - 1))); }

// The row of a sequence, and the head of its group, that a packed row is.
__device__ __forceinline__ int row_in(const KvAttnArgs& g, int p) { return (int)g.by_group((uint32_t)p); }
__device__ __forceinline__ int head_in(const KvAttnArgs& g, int p) { return p - row_in(g, p) * g.group; }

// The first slot of a sequence's tiles. A sequence of n packed rows behind r others
// has floor((r + n + (tile - 1) (s + 1)) / tile) - floor((r + (tile - 1) s) / tile) of
// them, at least ceil(n / tile), so that a slot's sequence is found by search
// and no list of tiles is made.
template <int TILE>
__device__ __forceinline__ long long tile_slot(const KvAttnArgs& g, int row, int s) {
  return ((long long)row * g.group + (long long)(TILE - 1) * s) / TILE;
}

// ln of a sum of weights relative to m (log2 units).
template <int KV>
__device__ __forceinline__ float lse_of(float m, float sum) {
  return sum == 0.f ? -INFINITY : (m - kShift<KV> + __builtin_amdgcn_logf(sum)) * kLn2;
}

// A sum times a factor that is not 0 but may have become it: an infinity stays.
__device__ __forceinline__ float scaled(float x, float f) { return fabsf(x) == INFINITY ? x : x * f; }

// Infinities and NaN. A weight of 0, or a zero part of a query, times one of them
// leaves a NaN, so whatever needs care shows in O, and no main loop looks for it.
// A wave takes rows whose sums are not finite again with redo_rows: without the
// keys whose K holds one, and with zeros in the place of those in V. careful_rows
// adds both, to the rows that see them, as the formula has it.
// Whether one of the n 16-byte units of a row of K or V holds one.
template <int KV>
__device__ __forceinline__ bool row_odd(const uint8_t* row, int n) {
  uint32_t odd = 0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const u32x4 w = *(const u32x4*)(row + 16 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (KV == KV_E4M3) {
        odd |= ((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;   // a byte of 0x7f
      } else {
        constexpr uint32_t M = KV == KV_F16 ? 0x7c00u : 0x7f80u;
        odd |= (uint32_t)((w[e] & M) == M) | (uint32_t)((w[e] & (M << 16)) == M << 16);
      }
    }
  }
  return odd != 0;
}

// R packed rows of a wave over the keys of [u0, u1) with such values, 64 at a time, in
// f32: for the scores a lane has a key, for the sums values of the head. Where K
// holds one the key is taken whole; of other keys the infinities and NaN of V alone, which
// have a weight above 0 whatever it is. A row whose query is not finite (lost) takes
// all keys whole, and here only. The sums are those of values d0 to d0 + DW - 1. Of an axis that waves share in strips of 32 keys,
// STEP apart, the wave has the strips from u0 on; strip i can hold such a key only
// if bit i >> shift of marks is set.
template <int KV, int DP, int DW, class T, int STEP, int R>
__device__ __forceinline__ void careful_rows(const KvAttnArgs& g, int s, const KvSeq& sq, const Span& sp, int u0, int u1, int kvh, uint64_t marks,
                                             int shift, int d0, const int (&p)[R], float (&o)[R][DW / 64], float (&m)[R], float (&l)[R],
                                             bool (&lost)[R]) {
  constexpr int N = DP / 64, NV = DW / 64, ES = KV == KV_E4M3 ? 1 : 2;
  const int lane = threadIdx.x & 63, D = g.kv.dim;
  float q[R][N];
  int pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row_in(g, p[r]);
    const T* src = (const T*)g.q + (sq.first + row) * g.ldq + (long long)(kvh * g.group + head_in(g, p[r])) * D;
    pos[r] = sq.len - sq.rows + row;
    m[r] = -INFINITY;
    l[r] = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      q[r][i] = (float)src[min(lane + 64 * i, D - 1)];
      odd |= !(fabsf(q[r][i]) < INFINITY);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) o[r][i] = 0.f;
    lost[r] = __ballot(odd) != 0;
    if (lost[r]) marks = ~0ull;
  }
#pragma unroll 1
  for (int base = u0, i = 0; base < u1; base += 2 * STEP, i += 2) {
    if (((marks >> (i >> shift) | marks >> min((i + 1) >> shift, 63)) & 1) == 0) continue;
    const int u = base + lane / 32 * STEP + lane % 32, key = u < sp.a ? u : sp.lo + u - sp.a;
    KvPlace at{};
    bool ok = u < u1 && (u >= sp.a || u < sp.sink);
    if (ok) ok = kv_place(g.kv, s, key, &at);
    if (!ok) at = KvPlace{0, 0};
    const long long off = kv_offset(g.kv, at, kvh) * ES;
    const uint8_t* kp = (const uint8_t*)g.kv.k + off;
    float ks = 1.f, vs = 1.f;
    if constexpr (KV == KV_E4M3) {
      ks = g.kv.k_scale[kv_scale_at(g.kv, at, kvh)];
      vs = g.kv.v_scale[kv_scale_at(g.kv, at, kvh)];
    }
    const bool k_odd = row_odd<KV>(kp, D * ES / 16) || !(ks < INFINITY), v_odd = row_odd<KV>((const uint8_t*)g.kv.v + off, D * ES / 16) || !(vs < INFINITY);
    bool sees[R], some = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sees[r] = ok && (k_odd || v_odd || lost[r]) && key <= pos[r] && (g.window == 0 || key > pos[r] - g.window || key < g.sinks);
      some |= sees[r];
    }
    const uint64_t any = __ballot(some);
    if (any == 0) continue;
    // eight sums, each of every eighth product
    float x[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[r][e] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll 1
      for (int d = 0; d < 64 && 64 * i + d < D; d += 8) {
        float k[8];
        if constexpr (KV == KV_E4M3) {
          const uint2 w = *(const uint2*)(kp + 64 * i + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t t = e < 4 ? w.x : w.y;
            k[e] = e % 4 == 0 ? __builtin_amdgcn_cvt_f32_fp8(t, 0) : e % 4 == 1 ? __builtin_amdgcn_cvt_f32_fp8(t, 1)
                   : e % 4 == 2 ? __builtin_amdgcn_cvt_f32_fp8(t, 2) : __builtin_amdgcn_cvt_f32_fp8(t, 3);
          }
        } else {
          const u32x4 w = *(const u32x4*)(kp + 2 * (64 * i + d));
#pragma unroll
          for (int e = 0; e < 8; ++e) k[e] = e % 2 == 0 ? value_lo<KV>(w[e / 2]) : value_hi<KV>(w[e / 2]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[r][e] = fmaf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, q[r][i]), d + e)), k[e], x[r][e]);
      }
    float w[R];
    uint64_t seen[R], slight[R];   // slight: a weight that is 0 here, but one for an infinity
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float t = (((x[r][0] + x[r][1]) + (x[r][2] + x[r][3])) + ((x[r][4] + x[r][5]) + (x[r][6] + x[r][7]))) * g.scale2 * ks;
      const bool whole = k_odd || lost[r];
      if (!sees[r] || !whole) t = -INFINITY;
      const float top = fmaxf(m[r], gg::wave_max(t)), f = top == m[r] ? 1.f : __builtin_amdgcn_exp2f(m[r] - top);
      m[r] = top;
      // a NaN or +inf leaves nothing of the row: e^(s - m) is a NaN with either
      w[r] = t == -INFINITY ? 0.f : t < INFINITY ? __builtin_amdgcn_exp2f(t - top) * (float)(1 << (int)kShift<KV>) : NAN;
      l[r] = f * l[r] + gg::wave_sum(w[r]);
#pragma unroll
      for (int i = 0; i < NV; ++i) o[r][i] = scaled(o[r][i], f);
      seen[r] = __ballot(sees[r]);
      slight[r] = __ballot(sees[r] && (!whole || (t > -INFINITY && w[r] == 0.f)));
    }
#pragma unroll 1
    for (uint64_t left = any; left; left &= left - 1) {
      const int b = __builtin_ctzll(left);
      const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)off, b), hi = (uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), b);
      const uint8_t* vp = (const uint8_t*)g.kv.v + (long long)(((uint64_t)hi << 32) | lo);
      float v[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int d = min(d0 + lane + 64 * i, D - 1);
        if constexpr (KV == KV_E4M3)
          v[i] = __builtin_amdgcn_cvt_f32_fp8((uint32_t)vp[d], 0) * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), b));
        else
          v[i] = value_lo<KV>((uint32_t)((const uint16_t*)vp)[d]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (((seen[r] >> b) & 1) == 0) continue;
        const float wr = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w[r]), b));
        const float wi = (slight[r] >> b) & 1 ? 1.f : wr;
#pragma unroll
        for (int i = 0; i < NV; ++i) o[r][i] = fmaf(fabsf(v[i]) < INFINITY ? wr : wi, v[i], o[r][i]);
      }
    }
  }
}

// The 16 packed rows from p0 on, those of `which` for certain, over the strips of
// 32 keys from u0 on, STEP apart, values d0 to d0 + DW - 1 of them: one wave, K and V
// straight from memory. Lane (c, quad) gets values d0 + 16 t + 4 quad + i of packed
// row c, its m and its sums of weights. buf: four rows of DW floats, ld apart, of the
// wave's own. The registers that a call of it saves are scratch memory, of 8192
// waves for each hardware queue in use: with 128 values at a time 0.19 GB, with all 256
// 0.45, and 0.87 with queries and V held too (windowed f32 turns; 64 at a time
// 0.08, but twice the time). It shares nothing with the other waves: with one NaN that
// all rows see, 61 tokens of 32 heads of 128 on 8 at up to 8192 positions take 323 us
// for 228, 2048 rows at 32768, 4 heads of 256 on 1, 6.1 ms for 0.33.
constexpr int kRedoDims = 128;
template <int KV, int DP, class T, int STEP, int DW = DP < kRedoDims ? DP : kRedoDims>
__device__ __forceinline__ void redo_rows(const KvAttnArgs& g, int s, const KvSeq& sq, const Span& sp, int u0, int u1, int kvh, int p0, uint32_t which,
                                          int d0, float* buf, int ld, f32x4 (&o)[DW / 16], float& m, float& l, float& le) {
  constexpr int NP = kParts<KV, T>, KC = DP / 32, VD = DW / 16, ES = KV == KV_E4M3 ? 1 : 2;
  const int lane = threadIdx.x & 63, c16 = lane & 15, quad = lane >> 4, D = g.kv.dim;
  const int p = min(p0 + c16, sq.rows * g.group - 1), row = row_in(g, p), pos = sq.len - sq.rows + row;
  const T* q = (const T*)g.q + (sq.first + row) * g.ldq + (long long)(kvh * g.group + head_in(g, p)) * D;
  const auto query = [&](int c, u32x4 (&qb)[NP]) __attribute__((always_inline)) {
    const int d = min(32 * c + 8 * quad, D - 8);
    const uint32_t on = 32 * c + 8 * quad < D ? ~0u : 0u;   // past D the query is 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[NP];
      split2<KV, NP>((float)q[d + 2 * i], (float)q[d + 2 * i + 1], w);
#pragma unroll
      for (int n = 0; n < NP; ++n) qb[n][i] = w[n] & on;
    }
  };
#pragma unroll
  for (int t = 0; t < VD; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  m = -INFINITY;
  l = le = 0.f;
  const auto of_lane = [](float x, int i) __attribute__((always_inline)) { return __shfl(x, i, 64); };
  // whether one of two 16-bit values is an infinity or a NaN
  const auto odd2 = [](uint32_t w) __attribute__((always_inline)) {
    constexpr uint32_t M = KV == KV_F16 ? 0x7c00u : 0x7f80u;
    return (uint32_t)((w & M) == M) | (uint32_t)((w & (M << 16)) == M << 16) << 1;
  };
  uint64_t marks = 0;
  int shift = 0, strip = 0;
  while (((u1 - u0) / STEP) >> shift > 63) ++shift;
#pragma unroll 1
  for (int u = u0; u < u1; u += STEP, ++strip) {
    const int x = u + (lane & 31), mine = x < sp.a ? x : sp.lo + x - sp.a;
    KvPlace at{};
    bool ok = x < u1 && (x >= sp.a || x < sp.sink);
    if (ok) ok = kv_place(g.kv, s, mine, &at);
    if (!ok) at = KvPlace{0, 0};
    const long long off = kv_offset(g.kv, at, kvh) * ES;
    float sk = 1.f, sv = 1.f;
    if constexpr (KV == KV_E4M3) {
      sk = g.kv.k_scale[kv_scale_at(g.kv, at, kvh)];
      sv = g.kv.v_scale[kv_scale_at(g.kv, at, kvh)];
    }
    const uint32_t placed = (uint32_t)__ballot(ok);
    uint32_t odd = (uint32_t)__ballot(!(sk < INFINITY));   // keys whose K holds an infinity or a NaN
    bool mark = !(sv < INFINITY);
    f32x4 sc[2];
    uint32_t k_odd[2] = {};
    const uint8_t* kp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
      kp[h] = (const uint8_t*)g.kv.k + __shfl(off, c16 + 16 * h, 64);
    }
    // the queries' parts are made again each time, for their registers
#pragma unroll 2
    for (int c = 0; c < KC; ++c) {
      const int d = min(32 * c + 8 * quad, D - 8);
      u32x4 qb[NP];
      query(c, qb);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 ka;
        if constexpr (KV == KV_E4M3) {
          const uint2 w = *(const uint2*)(kp[h] + d);
          ka[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.f, false));
          ka[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.f, true));
          ka[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.f, false));
          ka[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.f, true));
        } else {
          ka = *(const u32x4*)(kp[h] + 2 * d);
        }
        k_odd[h] |= odd2(ka[0]) | odd2(ka[1]) | odd2(ka[2]) | odd2(ka[3]);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) sc[h] = mfma16<KV>(ka, qb[n], sc[h]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint64_t b = __ballot(k_odd[h] != 0);
      b |= b >> 32;
      odd |= (uint32_t)((b | (b >> 16)) & 0xffff) << (16 * h);
    }
    const uint32_t live = placed & ~odd;
    mark |= (odd & placed) != 0;
    // this lane's keys are 4 quad + j and, from j = 4 on, 12 more
    const int key0 = u < sp.a ? u : sp.lo + u - sp.a;
    float y[8], mx = -INFINITY;
    uint32_t pb[NP][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 4 * quad + (j & 3) + 16 * (j >> 2), key = key0 + i;
      const bool sees = ((live >> i) & 1) && key <= pos && (g.window == 0 || key > pos - g.window || key < g.sinks);
      float t = sc[j >> 2][j & 3] * g.scale2;
      if constexpr (KV == KV_E4M3) t *= of_lane(sk, i);
      y[j] = sees ? t : -INFINITY;
      mx = fmaxf(mx, y[j]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // (no slack: with large values no weight is above 1)
    const float top = fmaxf(m, mx), f = top == m ? 1.f : __builtin_amdgcn_exp2f(m - top), ref = (top == -INFINITY ? 0.f : top) - kShift<KV>;
    m = top;
    l *= f;
    le *= f;
#pragma unroll
    for (int t = 0; t < VD; ++t) o[t] *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float w0 = __builtin_amdgcn_exp2f(y[2 * i] - ref), w1 = __builtin_amdgcn_exp2f(y[2 * i + 1] - ref);
      uint32_t w[NP];
      le += w0 + w1;
      split2<KV, NP>(w0, w1, w);
      if constexpr (NP == 1) {
        w0 = value_lo<KV>(w[0]);
        w1 = value_hi<KV>(w[0]);
      }
      l += w0 + w1;
      if constexpr (KV == KV_E4M3) {
        const int j = 4 * quad + (2 * i & 3) + 16 * (i >> 1);
        const float s0 = of_lane(sv, j), s1 = of_lane(sv, j + 1);
        w0 = s0 < INFINITY ? w0 * s0 : 0.f;
        w1 = s1 < INFINITY ? w1 * s1 : 0.f;
        split2<KV, NP>(w0, w1, w);
      }
#pragma unroll
      for (int n = 0; n < NP; ++n) pb[n][i] = w[n];
    }
    const uint8_t* vp[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) vp[j] = (const uint8_t*)g.kv.v + __shfl(off, 4 * quad + (j & 3) + 16 * (j >> 2), 64) + min(c16, D - 1) * ES;
#pragma unroll
    for (int t = 0; t < VD; ++t) {
      const int d = min(d0 + 16 * t, D - 16) * ES;   // what lies past D is nobody's
      u32x4 va;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t *r0 = vp[2 * i] + d, *r1 = vp[2 * i + 1] + d;
        if constexpr (KV == KV_E4M3) va[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)*r0 | ((uint32_t)*r1 << 8), 1.f, false));
        else va[i] = (uint32_t)*(const uint16_t*)r0 | ((uint32_t)*(const uint16_t*)r1 << 16);
        const uint32_t no = odd2(va[i]);
        mark |= no != 0;
        va[i] &= (no & 1 ? 0u : 0xffffu) | (no & 2 ? 0u : 0xffff0000u);
      }
#pragma unroll
      for (int n = NP - 1; n >= 0; --n) o[t] = mfma16<KV>(va, u32x4{pb[n][0], pb[n][1], pb[n][2], pb[n][3]}, o[t]);
    }
    if (__ballot(mark) != 0) marks |= 1ull << (strip >> shift);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  le += __shfl_xor(le, 16, 64);
  le += __shfl_xor(le, 32, 64);
  // the keys left out, four rows at a time
  constexpr int R = 4;
#pragma unroll 1
  for (uint32_t left = which; left;) {
    int c[R], pr[R], r_of = -1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      c[r] = left ? __builtin_ctz(left) : c[0];
      r_of = left && c16 == c[r] ? r : r_of;
      left &= left - 1;
      pr[r] = p0 + c[r];
    }
    float os[R][DW / 64], ms[R], ls[R], m2 = 0.f, l2 = 0.f;
    bool lost[R], drop = false;
    careful_rows<KV, DP, DW, T, STEP, R>(g, s, sq, sp, u0, u1, kvh, marks, shift, d0, pr, os, ms, ls, lost);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < DW / 64; ++i) buf[r * ld + lane + 64 * i] = os[r][i];
      m2 = r_of == r ? ms[r] : m2;
      l2 = r_of == r ? ls[r] : l2;
      drop = r_of == r ? lost[r] : drop;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (r_of >= 0) {
      if (drop) m = -INFINITY;
      const float top = fmaxf(m, m2), f = drop ? 0.f : m == top ? 1.f : __builtin_amdgcn_exp2f(m - top),
                  f2 = m2 == top ? 1.f : __builtin_amdgcn_exp2f(m2 - top);
      m = top;
      l = (drop ? 0.f : l * f) + l2 * f2;
      le = (drop ? 0.f : le * f) + l2 * f2;
#pragma unroll
      for (int t = 0; t < VD; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = (drop ? 0.f : o[t][i] * f) + scaled(buf[r_of * ld + 16 * t + 4 * quad + i], f2);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---------------------------------------------------------------------------
// Few rows: a block takes 16 packed rows of a K/V head and a chunk of keys, its
// waves 32 keys at a time in turn. K and V go from memory to registers, K in
// operand order as it lies, V in rows (16 lanes share one) and transposed by
// byte permutes: no barrier in the loop, and through LDS only where a step's rows lie
// and 8-bit rows' scales; the next step's K is asked for
// when this one's is used up, V likewise. Memory bounds it: 61 tokens of 32 heads of 128
// on 8 at up to 8192 positions 221 us and 7 more for the join, 5.4 TB/s; 3 tokens
// at up to 131072, 8-bit heads of 256, 138 and 5 us, 5.3 TB/s. Of one token's 8 us
// 1.3 go until the table is read, 2.8 until K and V are here, 2 for the two
// products and the weights, 1 to add the waves' sums.
// ---------------------------------------------------------------------------
template <int KV, int DP, class T>
__global__ __launch_bounds__(256, (DP <= 128 || (KV == KV_E4M3 && kParts<KV, T> == 1) ? 2 : 1)) void k_attn_few(KvAttnArgs g, int slot0, int slots) {
  constexpr int NP = kParts<KV, T>, KC = DP / 32, VD = DP / 16, OP = DP + 4;
  constexpr int ES = KV == KV_E4M3 ? 1 : 2;                 // bytes of an element in the pages
  constexpr int KL = KV == KV_E4M3 ? KC / 2 : KC, VW = VD * ES / 4;   // 16-byte loads of a K row, dwords of a V row
  __shared__ __align__(16) float o_all[4][kKvFewTile][OP];
  __shared__ float m_all[4][kKvFewTile], l_all[4][kKvFewTile], e_all[4][kKvFewTile];
  __shared__ __align__(16) long long key_off[4][32];        // where a step's rows lie, -1: nowhere
  __shared__ __align__(16) float k_sc[4][32], v_sc[4][32];
  __shared__ u32x4 q_all[NP][KC][64];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, quad = lane >> 4, D = g.kv.dim;
  // Heads fastest. With many tiles the chunks of one lie next to each other, and
  // a place further round for each: the eight XCDs take blocks in turn, and
  // without the turn one of them may get all of the last chunks, which few
  // sequences have (61 tokens at up to 8192, 8 chunks, 8 heads: 295 us, 229 so, 252
  // with the chunks slowest). With few tiles the chunks are slowest, so that the
  // last blocks are short ones (3 tokens at up to 131072, 8 heads: 155 us, 191 the other way).
  const int each = g.splits * g.kv.n_kv;
  int split, kvh, slot;
  if ((long long)slots * g.kv.n_kv >= 128) {
    const int tile = (int)(blockIdx.x / each), r = (int)((blockIdx.x % each + (uint32_t)tile) % each);
    kvh = r % g.kv.n_kv;
    split = r / g.kv.n_kv;
    slot = slot0 + tile;
  } else {
    const int r = (int)(blockIdx.x / g.kv.n_kv);
    kvh = (int)(blockIdx.x % g.kv.n_kv);
    split = r / slots;
    slot = slot0 + r % slots;
  }
  // beside k_attn_many only short sequences count, of a few tiles each
  const bool all = g.few_rows == 0x7fffffff;
  KvSeq sq;
  int s = slot / kKvFewTiles;
  if (all) s = kv_find(g.kv, slot, [&](int r, int i) { return tile_slot<kKvFewTile>(g, r, i); }, &sq);
  else sq = kv_seq(g.kv, s);
  if (s < 0) return;
  const long long tile_l = all ? slot - tile_slot<kKvFewTile>(g, sq.first, s) : slot % kKvFewTiles;
  const int packed = sq.rows * g.group;
  if (tile_l < 0 || tile_l * kKvFewTile >= packed || packed > g.few_rows) return;
  const int p0 = (int)tile_l * kKvFewTile;
  const Span sp = kv_span<32>(g, sq, row_in(g, p0), min(row_in(g, p0 + kKvFewTile - 1), sq.rows - 1));
  const int u0 = split * g.chunk, u1 = min(sp.n, u0 + g.chunk);
  if (split > 0 && u0 >= sp.n) return;
  const bool joined = sp.n > g.chunk;

  // this lane's packed row
  const int p = p0 + c16;
  const int pos = p < packed ? sq.len - sq.rows + row_in(g, p) : -1;
  const int pos_min = sq.len - sq.rows + row_in(g, p0), pos_max = sq.len - sq.rows + min(row_in(g, p0 + kKvFewTile - 1), sq.rows - 1);
  f32x4 o[VD];
#pragma unroll
  for (int t = 0; t < VD; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f, le = 0.f;   // le: of the weights before they are rounded, for lse
  typedef uint32_t vw_t __attribute__((ext_vector_type(VW > 4 ? 4 : VW)));
  constexpr int VN = VW > 4 ? VW / 4 : 1;
  u32x4 kr[2][KL];
  vw_t vr[8][VN];

  // The page of a step's keys, one a lane, is asked for a step before its places
  // are worked out and handed over in LDS; so are 8-bit rows' scales.
  int page = 0;
  float sk = 0.f, sv = 0.f;
  const int key_lane = lane & 31;
  auto ask = [&](int u) __attribute__((always_inline)) {
    const int x = u + key_lane, key = min(max(x < sp.a ? x : sp.lo + x - sp.a, 0), g.kv.places - 1);
    page = g.kv.table[(long long)s * g.kv.table_ld + (int)g.kv.page_div((uint32_t)key)];
  };
  uint32_t live = 0;   // bit i: key i of the step has a place; others are read from row 0
  auto places = [&](int u) __attribute__((always_inline)) {
    const int x = u + key_lane, key = x < sp.a ? x : sp.lo + x - sp.a;
    const bool ok = x < u1 && (x >= sp.a || x < sp.sink) && (uint32_t)page < (uint32_t)g.kv.n_pages;
    const KvPlace at{ok ? page : 0, ok ? key - (int)g.kv.page_div((uint32_t)key) * g.kv.page_size : 0};
    if (lane < 32) key_off[wv][lane] = kv_offset(g.kv, at, kvh) * ES;
    live = (uint32_t)__ballot(ok);
    if constexpr (KV == KV_E4M3) {
      sk = g.kv.k_scale[kv_scale_at(g.kv, at, kvh)];
      sv = g.kv.v_scale[kv_scale_at(g.kv, at, kvh)];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  const int dk = 16 / ES * quad, dv = VD * c16;
  const uint8_t* k_lane = (const uint8_t*)g.kv.k + dk * ES;
  const uint8_t* v_lane = (const uint8_t*)g.kv.v + (dv < D ? dv : 0) * ES;
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* r = k_lane + key_off[wv][16 * h + c16];
#pragma unroll
      for (int c = 0; c < KL; ++c) {
        const int d = 64 / ES * c;   // past D the query is 0
        kr[h][c] = *(const u32x4*)(r + (d + dk < D ? d * ES : -dk * ES));
      }
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* r = v_lane + key_off[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
#pragma unroll
      for (int n = 0; n < VN; ++n) vr[j][n] = ((const vw_t*)r)[n];
    }
  };

  // The first step's keys are asked for before the queries are made operands, of
  // which each wave makes a share for all (one token at 2049 positions, heads of
  // 256, both launches: 13.4 us where each wave made all of them first, 11.9 so).
  const int first = u0 + 32 * wv;
  ask(first);
  constexpr int QN = KC < 4 ? 1 : KC / 4;   // chunks of a wave
  typedef T q8_t __attribute__((ext_vector_type(8)));
  q8_t q8[QN];
  int q_at[QN];
  const bool q_wave = wv * QN < KC;
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int c = q_wave ? wv * QN + i : 0;
    // a lane's values of a chunk; with 8 bits those of two chunks lie together in K
    q_at[i] = KV == KV_E4M3 ? 64 * (c / 2) + 16 * quad + 8 * (c % 2) : 32 * c + 8 * quad;
    const int pr = min(p, packed - 1);
    const T* q = (const T*)g.q + (sq.first + row_in(g, pr)) * g.ldq + (long long)(kvh * g.group + head_in(g, pr)) * D + (q_at[i] < D ? q_at[i] : 0);
    if (g.q_vec) {
      constexpr int V = 16 / sizeof(T);
      typedef T vec_t __attribute__((ext_vector_type(V)));
      if constexpr (V == 8) {
        q8[i] = *(const vec_t*)q;
      } else {
        const vec_t lo = *(const vec_t*)q, hi = *(const vec_t*)(q + 4);
        q8[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) q8[i][k] = q[k];
    }
  }
  // (by waves without keys too, which read row 0: loads in a branch would all be
  // waited for behind it)
  places(first);
  ask(first + 128);
  load_k();
  load_v();
  if (q_wave) {
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const bool on = p < packed && q_at[i] < D;
      u32x4 part[NP];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t w[NP];
        split2<KV, NP>(on ? (float)q8[i][2 * k] : 0.f, on ? (float)q8[i][2 * k + 1] : 0.f, w);
#pragma unroll
        for (int n = 0; n < NP; ++n) part[n][k] = w[n];
      }
#pragma unroll
      for (int n = 0; n < NP; ++n) q_all[n][wv * QN + i][lane] = part[n];
    }
  }
  // for LDS only: a full barrier, or an acquire fence, would wait for the loads
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  u32x4 qb[NP][KC];
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int c = 0; c < KC; ++c) qb[n][c] = q_all[n][c][lane];

  // All of this wave's keys. (Not written in line: the weights are then compiled
  // into blocks of their own, 3 tokens at up to 131072, 8-bit heads of 256, 145.6 us for 142.4.)
  auto pass = [&]() __attribute__((always_inline)) {
  float ks[8], vs[8];
  // (left from the middle: a path around the last loads back to the start would
  // make K wait for V there)
  if (first < u1) for (int u = first;; u += 128) {
    if constexpr (KV == KV_E4M3) {
      if (lane < 32) {
        k_sc[wv][lane] = sk;
        v_sc[wv][lane] = sv;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ks[j] = k_sc[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
        vs[j] = v_sc[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
      }
    }
    // this lane's keys are 4 quad + j and, from j = 4 on, 12 more
    const uint32_t mine = __builtin_amdgcn_readfirstlane(live) >> (4 * quad);
    const bool miss = __builtin_amdgcn_readfirstlane(live) != 0xffffffffu;
    // S^T: 32 keys x 16 packed rows
    // with several parts in two sums each, chains of half the length
    constexpr int CHAINS = NP > 1 ? 2 : 1;
    f32x4 sc[2], acc[CHAINS][2];
#pragma unroll
    for (int i = 0; i < CHAINS; ++i) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      u32x4 ka[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (KV == KV_E4M3) {
          typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
          const uint32_t k0 = kr[h][c / 2][2 * (c % 2)], k1 = kr[h][c / 2][2 * (c % 2) + 1];
          const bf16x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k0, 1.f, false),
                       a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k0, 1.f, true),
                       a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k1, 1.f, false),
                       a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k1, 1.f, true);
          ka[h] = u32x4{__builtin_bit_cast(uint32_t, a0), __builtin_bit_cast(uint32_t, a1), __builtin_bit_cast(uint32_t, a2),
                        __builtin_bit_cast(uint32_t, a3)};
        } else {
          ka[h] = kr[h][c];
        }
      }
#pragma unroll
      for (int k = NP - 1; k >= 0; --k)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[c % CHAINS][h] = mfma16<KV>(ka[h], qb[k][c], acc[c % CHAINS][h]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = acc[0][h];
      if constexpr (CHAINS > 1) sc[h] += acc[CHAINS - 1][h];
    }
    const int next = u + 128;
    if (next < u1) {
      places(next);
      ask(next + 128);
      load_k();
    }
    // scores in log2 units; what the row does not see is -inf
    const int key0 = u < sp.a ? u : sp.lo + u - sp.a;
    float x[8], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = sc[j >> 2][j & 3] * g.scale2;
      if constexpr (KV == KV_E4M3) x[j] *= ks[j];
    }
    // most steps are seen whole by all rows
    const bool whole = !miss && key0 + 31 <= pos_min && (g.window == 0 || key0 > pos_max - g.window || key0 + 31 < g.sinks);
    uint32_t here = ~0u;   // bit j: the row sees key j
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = (j & 3) + 16 * (j >> 2), key = key0 + 4 * quad + i;
        const bool sees = ((mine >> i) & 1) && key <= pos && (g.window == 0 || key > pos - g.window || key < g.sinks);
        x[j] = sees ? x[j] : -INFINITY;
        here = sees ? here : here & ~(1u << j);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, x[j]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    float f = 1.f;
    if (__ballot(mx > m + kSlack)) {
      const float mn = mx > m + kSlack ? mx : m;
      f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
      le *= f;
#pragma unroll
      for (int t = 0; t < VD; ++t) o[t] *= f;
    }
    const float ref = (m == -INFINITY ? 0.f : m) - kShift<KV>;
    // weights, as the second product's operand
    u32x4 pb[NP];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float w0 = __builtin_amdgcn_exp2f(x[2 * i] - ref), w1 = __builtin_amdgcn_exp2f(x[2 * i + 1] - ref);
      uint32_t w[NP];
      le += w0 + w1;
      if constexpr (NP == 1) {
        // out is divided by the sum of the rounded weights: their errors cancel where they are alike
        if constexpr (KV == KV_F16) w[0] = pack_f16(w0, w1);
        else w[0] = pack_bf16(w0, w1);
        w0 = value_lo<KV>(w[0]);
        w1 = value_hi<KV>(w[0]);
      }
      l += w0 + w1;
      if constexpr (KV == KV_E4M3) {
        w0 *= vs[2 * i];
        w1 *= vs[2 * i + 1];
        if (!whole) {   // a hidden row's scale may be a NaN
          w0 = (here >> (2 * i)) & 1 ? w0 : 0.f;
          w1 = (here >> (2 * i + 1)) & 1 ? w1 : 0.f;
        }
      }
      if constexpr (NP > 1 || KV == KV_E4M3) split2<KV, NP>(w0, w1, w);
#pragma unroll
      for (int k = 0; k < NP; ++k) pb[k][i] = w[k];
    }
    // V of keys that are not there counts as 0: what lies there may be a NaN
    if (miss) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int n = 0; n < VN; ++n) vr[j][n] = (mine >> ((j & 3) + 16 * (j >> 2))) & 1 ? vr[j][n] : (vw_t)0;
    }
    if constexpr (KV == KV_E4M3) {
      // bytes of two keys side by side, then converted: four values of a head
#pragma unroll
      for (int t = 0; t < VD; t += 4) {
        u32x4 va[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w0 = vr[2 * i][t / 16][t / 4 % 4], w1 = vr[2 * i + 1][t / 16][t / 4 % 4];
          const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400u), hi = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
          va[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
          va[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
          va[2][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
          va[3][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
        }
#pragma unroll
        for (int k = NP - 1; k >= 0; --k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t + e] = mfma16<KV>(va[e], pb[k], o[t + e]);
      }
    } else {
      constexpr int TS = NP > 1 ? 4 : 2;   // values at a time: sums that wait for each other lie TS instructions apart
#pragma unroll
      for (int t = 0; t < VD; t += TS) {
        u32x4 va[TS];
#pragma unroll
        for (int e = 0; e < TS; e += 2)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w0 = vr[2 * i][(t + e) / 8][(t + e) / 2 % 4], w1 = vr[2 * i + 1][(t + e) / 8][(t + e) / 2 % 4];
            va[e][i] = lower2(w0, w1);
            va[e + 1][i] = upper2(w0, w1);
          }
#pragma unroll
        for (int k = NP - 1; k >= 0; --k)
#pragma unroll
          for (int e = 0; e < TS; ++e) o[t + e] = mfma16<KV>(va[e], pb[k], o[t + e]);
      }
    }
    if (next >= u1) {
      asm volatile("");   // an exit of its own
      break;
    }
    load_v();
  }
  };
  pass();
  uint32_t again;   // rows whose sums are not finite
  {
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < VD; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = fmaf(o[t][i], 0.f, z[i]);
    uint64_t odd = __ballot((z[0] + z[1]) + (z[2] + z[3]) != 0.f && p < packed);   // 0 times an infinity or a NaN
    odd |= odd >> 32;
    again = (uint32_t)(odd | (odd >> 16)) & 0xffffu;
  }
  // (expected not to be: in line this code costs a single token 0.4 us)
  if (__builtin_expect(again != 0, 0)) {
    constexpr int DW = DP < kRedoDims ? DP : kRedoDims;
    float m2, l2, le2;
#pragma unroll 1
    for (int d0 = 0; d0 < DP; d0 += DW) {
      f32x4 o2[DW / 16];
      redo_rows<KV, DP, T, 128>(g, s, sq, sp, first, u1, kvh, p0, again, d0, &o_all[wv][0][d0], OP, o2, m2, l2, le2);
#pragma unroll
      for (int t = 0; t < DW / 16; ++t) *(f32x4*)&o_all[wv][c16][d0 + 16 * t + 4 * quad] = o2[t];
    }
    m = m2;
    l = quad == 0 ? l2 : 0.f;
    le = quad == 0 ? le2 : 0.f;
  }

  // the four waves' parts; this lane has values 4 VD quad + VD i + t of its packed row
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  le += __shfl_xor(le, 16, 64);
  le += __shfl_xor(le, 32, 64);
  if (lane < 16) {
    m_all[wv][lane] = m;
    l_all[wv][lane] = l;
    e_all[wv][lane] = le;
  }
  __syncthreads();
  {
    const float top = fmaxf(fmaxf(m_all[0][c16], m_all[1][c16]), fmaxf(m_all[2][c16], m_all[3][c16]));
    const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
    float* dst = &o_all[wv][c16][4 * VD * quad];
    if (__builtin_expect(again != 0, 0)) {   // they lie there
#pragma unroll 1
      for (int i = 0; i < 4 * VD; ++i) dst[i] = scaled(dst[i], f);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < VD; t += 4)
          *(f32x4*)(dst + VD * i + t) = f32x4{f * o[t][i], f * o[t + 1][i], f * o[t + 2][i], f * o[t + 3][i]};
    }
  }
  __syncthreads();
  for (int e = tid; e < kKvFewTile * (DP / 4); e += 256) {
    const int r = e / (DP / 4), d = 4 * (e % (DP / 4)), pr = p0 + r;
    if (pr >= packed || d >= D) continue;
    float top = m_all[0][r], sum = 0.f, exact = 0.f;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, m_all[w][r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = m_all[w][r] == top ? 1.f : __builtin_amdgcn_exp2f(m_all[w][r] - top);
      sum += f * l_all[w][r];
      exact += f * e_all[w][r];
    }
    f32x4 v = *(const f32x4*)&o_all[0][r][d];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += *(const f32x4*)&o_all[w][r][d];
    const long long orow = sq.first + row_in(g, pr);
    const int oh = kvh * g.group + head_in(g, pr);
    if (joined) {
      const long long at = ((long long)split * g.kv.n_rows + orow) * g.n_q + oh;
      *(f32x4*)(g.part_o + at * D + d) = v;
      if (d == 0) *(f32x4*)(g.part_ml + 4 * at) = f32x4{top, sum, exact, 0.f};
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T* out = (T*)g.out + orow * g.ldo + (long long)oh * D + d;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = (T)(v[i] * inv);
      if (d == 0 && g.lse) g.lse[orow * g.n_q + oh] = lse_of<KV>(top, exact);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: a block takes 128 packed rows of a K/V head, 32 a wave, and a chunk
// of keys, 64 at a time (32 with heads above 128 where rows are f32, or f16 on
// other than f16 pages, or pages 8-bit). The waves share K and V through
// LDS, two tiles of each: while one is used the next arrives by DMA, 1 KB of
// whole rows a copy, in the order of memory (16-byte units of a row at permuted
// places, the usual way to keep reads from meeting in a bank, take the copies
// twice as long here), at places such that neither the reads of K (a row a
// lane) nor those of V (transposed by the read, four rows to 16 lanes) meet in a
// bank. One barrier a tile. 8-bit rows go to a place of their wave's own, and from
// there as bf16 into one stage, between two barriers a tile: with bf16 rows and heads
// up to 128 that fits two blocks a CU, with 13 registers in scratch memory. (Two
// sequences of 2048 rows to 8192 positions, 16 heads of 128 on 4: 400 us; one
// block a CU with two stages, a barrier a tile, 599; loads to registers, which
// the compiler waits for too early, 989. bf16 pages take 319.)
// ---------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <int KV>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (KV == KV_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// The sum of two 16-bit weights and c.
template <int KV>
__device__ __forceinline__ float add2(uint32_t w, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (KV == KV_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{1, 1}, c, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
}
// A product that is rounded before what follows.
__device__ __forceinline__ float times(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
// One DMA instruction: lane l's 16 bytes at src go to dst + 16 l. Inline asm,
// because the compiler would wait for every copy in flight before any LDS read;
// the wait before the barrier that precedes the readers is written out.
__device__ __forceinline__ void dma16(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(src)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint64_t src, uint32_t dst) {   // lane l's four bytes
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(src)
               : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_at(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p; }

// What a key without a place is read from.
__device__ __attribute__((aligned(16))) const uint8_t kv_zeros[kKvMaxDim * 2] = {};
__device__ const float kv_one = 1.f;

// The rows of a wave of k_attn_many whose sums are not finite, 16 at a time. A
// call, and no reference among its arguments: in line its registers are taken from
// the main loop (prompts of 32 heads of 128 79 us for 77.5, windowed f32 turns 70.4 for 67.7).
// gp: the kernel's arguments where they lie.
typedef __attribute__((address_space(3))) float lds_float;
template <int KV, int DP, class T>
__device__ __attribute__((noinline)) void redo_many(const KvAttnArgs* gp, int s, int first, int rows, int len, int lo, int a, int sink, int n, int u0, int u1, int kvh,
                                                    int split, int pw, uint32_t again, uint32_t lds) {
  const auto uni = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };
  const uint64_t at = (uint32_t)uni((int)(uint32_t)(uintptr_t)gp) | (uint64_t)(uint32_t)uni((int)((uintptr_t)gp >> 32)) << 32;
  const KvAttnArgs& g = *(const KvAttnArgs*)(const __attribute__((address_space(4))) KvAttnArgs*)(uintptr_t)at;
  const KvSeq sq{uni(first), uni(rows), uni(len)};
  const Span sp{uni(lo), uni(a), uni(sink), uni(n)};
  s = uni(s), u0 = uni(u0), u1 = uni(u1), kvh = uni(kvh), split = uni(split), pw = uni(pw), again = uni(again), lds = uni(lds);
  const int lane = threadIdx.x & 63, D = g.kv.dim;
  const bool joined = sp.n > g.chunk;
#pragma unroll 1
  for (int h = 0; h < 32; h += 16) {
    const uint32_t which = (again >> h) & 0xffffu;
    if (which == 0) continue;
    constexpr int DW = DP < kRedoDims ? DP : kRedoDims;
    const int c16 = lane & 15, quad = lane >> 4, p2 = pw + h + c16;
#pragma unroll 1
    for (int d0 = 0; d0 < D; d0 += DW) {
      f32x4 o2[DW / 16];
      float m2, l2, le2;
      redo_rows<KV, DP, T, 32>(g, s, sq, sp, u0, u1, kvh, pw + h, which, d0, (float*)(lds_float*)(uintptr_t)lds, DW, o2, m2, l2, le2);
      if (((which >> c16) & 1) == 0) continue;
      const int orow = sq.first + row_in(g, p2), oh = kvh * g.group + head_in(g, p2);
      const long long to = ((long long)split * g.kv.n_rows + orow) * g.n_q + oh;
      const float inv = l2 == 0.f ? 0.f : 1.f / l2;
#pragma unroll
      for (int t = 0; t < DW / 16; ++t) {
        const int e = d0 + 16 * t + 4 * quad;
        if (d0 + 16 * t >= D) continue;
        if (joined) *(f32x4*)(g.part_o + to * D + e) = o2[t];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!joined) ((T*)g.out)[orow * g.ldo + (long long)oh * D + e + i] = (T)(o2[t][i] * inv);
      }
      if (quad == 0 && d0 == 0) {
        if (joined) *(f32x4*)(g.part_ml + 4 * to) = f32x4{m2, l2, le2, 0.f};
        else if (g.lse) g.lse[(long long)orow * g.n_q + oh] = lse_of<KV>(m2, le2);
      }
    }
  }
}

template <int KV, int DP, class T>
__global__ __launch_bounds__(256, (kParts<KV, T> > 1 || DP > 128 ? 1 : 2)) void k_attn_many(KvAttnArgs g, int slot0, int slots) {
  constexpr int NP = kParts<KV, T>, KT = DP == 256 && (NP > 1 || KV == KV_E4M3) ? 32 : 64, UN = DP / 8, RPI = 64 / UN, IPW = KT / RPI / 4;
  constexpr int KH = KT / 32, DT = DP / 32, CH = DP / 16, ES = KV == KV_E4M3 ? 1 : 2;
  // In LDS a copy's RPI rows are 1024 bytes, and some more to the next one: 16
  // for K, 32 for V. Scores take the keys of a tile in an order in which
  // neighbouring lanes read neighbouring copies: row m of 32 is key
  // RPI (m % NI) + m / NI.
  constexpr int NI = 32 / RPI, RB = DP * 2, KP = 1024 + 16, VP = 1024 + 32;
  constexpr bool RAW = KV == KV_E4M3;
  constexpr int STAGES = RAW ? 1 : 2, CP = RAW ? IPW / 2 : IPW;   // CP: copies of a wave, for K or V
  __shared__ __align__(16) uint8_t kbuf[STAGES][KT / RPI * KP], vbuf[STAGES][KT / RPI * VP];
  // 8-bit rows are copied as they are, each wave's to a place of its own, and
  // converted from there into the one stage of K and of V.
  __shared__ __align__(16) uint8_t kraw[RAW ? KT * DP : 16], vraw[RAW ? KT * DP : 16];
  __shared__ __align__(16) float scales[RAW ? 2 : 1][2][4][RAW ? 64 : 4];
  __shared__ __align__(16) float hole[2][KT];   // -inf where a key has no place
  __shared__ __align__(16) int holes[2][4];     // whether a wave's keys have any
  __shared__ __align__(16) long long row_off[2][KT];   // bytes from the pool's start to a row, -1: none
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, half = lane >> 5, D = g.kv.dim;
  // Blocks with one value of blockIdx % 8 share an XCD and its L2: they take a
  // contiguous range of an order with the tiles fastest, which read the same keys.
  const int G = gridDim.x, xcd = blockIdx.x & 7;
  const int unit = xcd * (G >> 3) + min(xcd, G & 7) + (blockIdx.x >> 3);
  const int slot = slot0 + unit % slots, ks_ = unit / slots;
  const int split = ks_ % g.splits, kvh = ks_ / g.splits;
  KvSeq sq;
  const int s = kv_find(g.kv, slot, [&](int r, int i) { return tile_slot<kKvManyTile>(g, r, i); }, &sq);
  if (s < 0) return;
  const long long tile_l = slot - tile_slot<kKvManyTile>(g, sq.first, s);
  const int packed = sq.rows * g.group;
  if (tile_l < 0 || tile_l * kKvManyTile >= packed || packed <= g.few_rows) return;
  const int p0 = (int)tile_l * kKvManyTile;
  const Span sp = kv_span<64>(g, sq, row_in(g, p0), min(row_in(g, p0 + kKvManyTile - 1), sq.rows - 1));
  const int u0 = split * g.chunk, u1 = min(sp.n, u0 + g.chunk);
  if (split > 0 && u0 >= sp.n) return;
  const bool joined = sp.n > g.chunk;
  const int before = sq.len - sq.rows;
  const int pw = p0 + 32 * wv;
  int p = pw + c32;
  const int pos = p < packed ? before + row_in(g, p) : -1;
  const bool active = pw < packed;   // this wave has rows
  const int pos_min = before + row_in(g, pw), pos_max = before + min(row_in(g, pw + 31), sq.rows - 1);

  // queries as operand columns; a negative scale turns their signs, so that the
  // largest product is the largest score, and scale 0 takes them out
  const float scale2 = g.scale2 == 0.f ? 1.f : fabsf(g.scale2), sign = g.scale2 > 0.f ? 1.f : g.scale2 < 0.f ? -1.f : 0.f;
  u32x4 qb[NP][CH];
  {
    const T* q = (const T*)g.q + (p < packed ? (sq.first + row_in(g, p)) * g.ldq + (long long)(kvh * g.group + head_in(g, p)) * D : 0);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int d = 16 * c + 8 * half;
      float f[8] = {};
      if (p < packed && d < D) {
        if (g.q_vec) {
          constexpr int V = 16 / sizeof(T);
          typedef T vec_t __attribute__((ext_vector_type(V)));
#pragma unroll
          for (int i = 0; i < 8; i += V) {
            const vec_t t = *(const vec_t*)(q + d + i);
#pragma unroll
            for (int k = 0; k < V; ++k) f[i + k] = sign * (float)t[k];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = sign * (float)q[d + i];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[NP];
        split2<KV, NP>(f[2 * i], f[2 * i + 1], w);
#pragma unroll
        for (int k = 0; k < NP; ++k) qb[k][c][i] = w[k];
      }
    }
  }

  // A wave copies RW rows of a tile; lane l's part of copy i is unit l % UN (in
  // LDS) of row (wv IPW + i) RPI + l / UN. Where the rows lie is found by a lane
  // each and handed over in LDS. Page ids are asked for a tile ahead and looked
  // at when its rows are fetched: waiting for one sooner would wait for the
  // copies before it too, and so would any branch or spill between the copies.
  constexpr int RW = KT / 4;
  const int tiles = (u1 - u0 + KT - 1) / KT;
  int page = 0;
  auto key_of = [&](int u) __attribute__((always_inline)) { return u < sp.a ? u : sp.lo + u - sp.a; };
  auto ask = [&](int t) __attribute__((always_inline)) {
    const int key = min(max(key_of(u0 + t * KT + wv * RW + lane % RW), 0), g.kv.places - 1);
    page = g.kv.table[(long long)s * g.kv.table_ld + (int)g.kv.page_div((uint32_t)key)];
  };
  auto rows = [&](int t) __attribute__((always_inline)) {
    const int r = wv * RW + lane % RW, x = u0 + t * KT + r, key = key_of(x);
    const bool ok = x < u1 && (x >= sp.a || x < sp.sink) && (uint32_t)page < (uint32_t)g.kv.n_pages;
    const KvPlace at{ok ? page : 0, ok ? key - (int)g.kv.page_div((uint32_t)key) * g.kv.page_size : 0};
    const long long off = kv_offset(g.kv, at, kvh) * ES;
    if (lane < RW) {
      row_off[t & 1][r] = ok ? off : -1;
      hole[t & 1][r] = ok ? 0.f : -INFINITY;
    }
    const int any = __ballot(!ok) != 0;
    if (lane == 0) holes[t & 1][wv] = any;
    if constexpr (KV == KV_E4M3) {
      const long long i = kv_scale_at(g.kv, at, kvh);
      dma4(ok ? (uint64_t)(uintptr_t)(g.kv.k_scale + i) : (uint64_t)(uintptr_t)&kv_one, lds_at(scales[t & 1][0][wv]));
      dma4(ok ? (uint64_t)(uintptr_t)(g.kv.v_scale + i) : (uint64_t)(uintptr_t)&kv_one, lds_at(scales[t & 1][1][wv]));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  // Sends for copy i of K or V of tile t: into its LDS stage, or its wave's place for 8-bit rows.
  constexpr int CU = 1024 / (DP * ES), CL = 64 / CU;   // rows of a copy, lanes to one
  auto fetch1 = [&](auto is_k, int t, int i) __attribute__((always_inline)) {
    const int st = t & 1, r = wv * RW + i * CU + lane / CL, unit = lane % CL;
    const long long off = row_off[st][r];
    const bool ok = off >= 0 && 16 / ES * unit < D;
    const uint64_t at = (uint64_t)(uintptr_t)(is_k ? g.kv.k : g.kv.v) + (uint64_t)off + (uint32_t)(16 * unit);
    const uint8_t* src = (const uint8_t*)(uintptr_t)(ok ? at : (uint64_t)(uintptr_t)kv_zeros);
    if constexpr (RAW) dma16(src, is_k ? lds_at(&kraw[(wv * CP + i) * 1024]) : lds_at(&vraw[(wv * CP + i) * 1024]));
    else dma16(src, is_k ? lds_at(&kbuf[st % STAGES][(wv * IPW + i) * KP]) : lds_at(&vbuf[st % STAGES][(wv * IPW + i) * VP]));
  };
  auto fetch = [&](auto is_k, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CP; ++i) fetch1(is_k, t, i);
  };
  // This wave's 8-bit rows of tile t, which have arrived, as bf16 into the stage.
  auto settle = [&](auto is_k, int t) __attribute__((always_inline)) {
    if constexpr (KV == KV_E4M3) {
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        const u32x4 w = *(const u32x4*)(is_k ? &kraw[(wv * CP + i) * 1024 + 16 * lane] : &vraw[(wv * CP + i) * 1024 + 16 * lane]);
        const int rw = i * CU + lane / CL, r = wv * RW + rw;
        const float sc = scales[t & 1][is_k ? 0 : 1][wv][rw];
        u32x4 o[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e / 2][2 * (e % 2)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e], sc, false));
          o[e / 2][2 * (e % 2) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e], sc, true));
        }
        uint8_t* dst = is_k ? &kbuf[0][r / RPI * KP + r % RPI * RB + 32 * (lane % CL)] : &vbuf[0][r / RPI * VP + r % RPI * RB + 32 * (lane % CL)];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *(u32x4*)(dst + 16 * e) = sc == sc ? o[e] : u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
      }
    }
  };
  constexpr std::true_type K{}, yes{};
  constexpr std::false_type V{}, no{};

  f32x16 o[DT], sc[KH];
  u32x4 pb[2 * KH][NP];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = -INFINITY, l = 0.f, le = 0.f;
  const int kbase = c32 % NI * KP + c32 / NI * RB + 16 * half;
  // V's lanes: four rows of 16 values to 16 lanes, those of the second half of a wave four rows on
  const int vm = 4 * half + ((lane & 15) >> 2), vbase = vm % NI * VP + vm / NI * RB + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  constexpr int V8 = 8 % NI * VP + 8 / NI * RB, V16 = 16 % NI * VP + 16 / NI * RB;   // rows m + 8, m + 16

  // Scores of tile t (QK) into sc, and (EX) the weights of what sc held before into
  // pb, each in the other's shadow, in the order written here: a slot is a read
  // of K four slots ahead, the matrix instructions of one operand, a share of the
  // weights and now and then a copy of V's next tile: sent in one go the copies
  // would hold the wave up until their addresses are through.
  constexpr int AHEAD = 4;
  auto scores = [&](auto QK, auto EX, int t) __attribute__((always_inline)) {
    constexpr int N = KH * CH, PAIRS = KH * 8;
    f32x16 nx[KH];
    const float ref = (m == -INFINITY ? 0.f : m) - kShift<KV>;
    const uint8_t* kst = kbuf[t % STAGES];
    u32x4 ka[N];
    auto read = [&](int c) __attribute__((always_inline)) {
      ka[c] = *(const u32x4*)&kst[kbase + c / CH * NI * KP + 32 * (c % CH)];
    };
    auto pair = [&](int e) __attribute__((always_inline)) {   // scores 2e and 2e + 1
      const int h = e / 8, i = e % 8;
      // f32: a product of its own, so that the reference's own key has weight 1
      const float s0 = sc[h][2 * i], s1 = sc[h][2 * i + 1];
      const float w0 = __builtin_amdgcn_exp2f(NP > 1 ? times(s0, scale2) - ref : fmaf(s0, scale2, -ref)),
                  w1 = __builtin_amdgcn_exp2f(NP > 1 ? times(s1, scale2) - ref : fmaf(s1, scale2, -ref));
      le += w0 + w1;
      uint32_t w[NP];
      split2<KV, NP>(w0, w1, w);
      if constexpr (NP == 1) l = add2<KV>(w[0], l);
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        asm volatile("" : "+v"(w[k]));   // here, not where it is used
        pb[e / 4][k][e % 4] = w[k];
      }
    };
    if constexpr (QK) {
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) nx[h][i] = 0.f;
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) read(c);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (c + AHEAD < N) read(c + AHEAD);
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) nx[c / CH] = mfma32<KV>(ka[c], qb[k][c % CH], nx[c / CH]);
        if constexpr (EX) {
#pragma unroll
          for (int e = c * PAIRS / N; e < (c + 1) * PAIRS / N; ++e) pair(e);
          if (c % (N / CP) == 0) fetch1(V, t, c / (N / CP));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int h = 0; h < KH; ++h) sc[h] = nx[h];
    } else {
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) pair(e);
    }
  };
  // What a row does not see gets -inf; then the largest score.
  int4 hs;   // whether tile t + 1 has keys without a place
  auto mask = [&](int t) __attribute__((always_inline)) {
    const int st = t & 1, key0 = key_of(u0 + t * KT), key1 = key0 + KT - 1;
    if (key1 > pos_min || (g.window > 0 && !(key0 > pos_max - g.window || key1 < g.sinks)) || (hs.x | hs.y | hs.z | hs.w) != 0) {
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int m = 8 * (i >> 2) + 4 * half + (i & 3), j = 32 * h + RPI * (m % NI) + m / NI, key = key0 + j;
          const bool sees = key <= pos && (g.window == 0 || key > pos - g.window || key < g.sinks) && hole[st][j] == 0.f;
          sc[h][i] = sees ? sc[h][i] : -INFINITY;
        }
    }
  };
  // O^T += V^T P^T of tile t; MX: the largest of the scores in sc meanwhile, and the
  // copies of K two tiles on.
  float mx = -INFINITY;
  auto products = [&](auto PV, auto MX, int t) __attribute__((always_inline)) {
    const uint8_t* vst = vbuf[t % STAGES];
    if constexpr (MX) mx = -INFINITY;
    if constexpr (PV) {
      constexpr int N = 2 * KH * DT;
      u32x4 va[N];
      auto read = [&](int c) __attribute__((always_inline)) {
        const uint8_t* src = &vst[vbase + c / DT / 2 * NI * VP + c / DT % 2 * V16 + 64 * (c % DT)];
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lds4;
        const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)lds_at(src)),
                    a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)lds_at(src + V8));
        const uint2 b0 = __builtin_bit_cast(uint2, a0), b1 = __builtin_bit_cast(uint2, a1);
        va[c] = u32x4{b0.x, b0.y, b1.x, b1.y};
      };
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) read(c);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (c + AHEAD < N) read(c + AHEAD);
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) o[c % DT] = mfma32<KV>(va[c], pb[c / DT][k], o[c % DT]);
        if constexpr (MX) {   // two scores a slot
#pragma unroll
          for (int e = c * KH * 8 / N; e < (c + 1) * KH * 8 / N; ++e)
            mx = fmaxf(fmaxf(mx, sc[e / 8][2 * (e % 8)]), sc[e / 8][2 * (e % 8) + 1]);
          if (c % (N / CP) == 0) fetch1(K, t + 2, c / (N / CP));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else if constexpr (MX) {
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[h][i]);
    }
    if constexpr (MX) mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * scale2;
  };
  auto rescale = [&]() __attribute__((always_inline)) {
    if (__ballot(mx > m + kSlack)) {
      const float mn = mx > m + kSlack ? mx : m;
      const float f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
      le *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
  };

  // K runs a tile ahead of V: while tile t's weights are made, the scores of
  // tile t + 1 are; the stage that a copy fills was last read before the barrier.
  // Tiles that a wave's rows do not see are taken all the same, masked: the
  // others would be waited for. K of tiles behind the last is read as zeros.
  if (tiles > 0) {
    const auto wait = []() __attribute__((always_inline)) { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
    ask(0);
    rows(0);
    ask(1);
    fetch(K, 0);
    fetch(V, 0);
    rows(1);
    ask(2);
    if constexpr (RAW) {
      wait();
      settle(K, 0);
      fetch(K, 1);
    } else {
      fetch(K, 1);
      wait();
    }
    __syncthreads();
    hs = *(const int4*)holes[0];
    scores(yes, no, 0);
    mask(0);
    products(no, yes, 0);
    rescale();
    for (int t = 0; t + 1 < tiles; ++t) {
      wait();            // this wave's copies of K t + 1 and V t
      __syncthreads();   // and everybody's; nobody reads the tiles before them any more
      hs = *(const int4*)holes[(t + 1) & 1];
      settle(K, t + 1);
      settle(V, t);
      rows(t + 2);
      ask(t + 3);
      if constexpr (RAW) __syncthreads();
      scores(yes, yes, t + 1);
      mask(t + 1);
      products(yes, yes, t);
      rescale();
    }
    wait();
    if constexpr (RAW) {
      __syncthreads();
      settle(V, tiles - 1);
    }
    __syncthreads();
    scores(no, yes, tiles - 1);
    products(yes, no, tiles - 1);
  }
  if (!active) return;

  asm volatile("" : "+v"(p));   // what follows from it is worked out here: it need not be kept in the loop
  const int row = sq.first + row_in(g, p), head = kvh * g.group + head_in(g, p);
  l += __shfl_xor(l, 32, 64);
  le += __shfl_xor(le, 32, 64);
  if constexpr (NP > 1) l = le;
  float z = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) z = fmaf(o[d][i], 0.f, z);
  uint64_t again = __ballot(z != 0.f && p < packed);   // 0 times an infinity or a NaN
  again |= again >> 32;
  const bool mine = (again >> c32) & 1;
  const long long at = ((long long)split * g.kv.n_rows + row) * g.n_q + head;
  if (p < packed && !mine) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = (T*)g.out + row * g.ldo + (long long)head * D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 32 * d + 8 * i + 4 * half;
        if (e >= D) continue;
        const f32x4 v = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (joined) {
          *(f32x4*)(g.part_o + at * D + e) = v;
        } else if (g.out_vec) {
          typedef T vec_t __attribute__((ext_vector_type(4)));
          *(vec_t*)(out + e) = vec_t{(T)(v[0] * inv), (T)(v[1] * inv), (T)(v[2] * inv), (T)(v[3] * inv)};
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) out[e + k] = (T)(v[k] * inv);
        }
      }
    if (half == 0) {
      if (joined) *(f32x4*)(g.part_ml + 4 * at) = f32x4{m, l, le, 0.f};
      else if (g.lse) g.lse[(long long)row * g.n_q + head] = lse_of<KV>(m, le);
    }
  }
  // the others; K's stages, which nobody reads any more, have a place for each wave
  static_assert(sizeof(kbuf) >= 4 * 4 * DP * sizeof(float), "four rows for each of four waves");
  if (__builtin_expect(again != 0, 0))
    redo_many<KV, DP, T>((const KvAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr(), s, sq.first, sq.rows, sq.len, sp.lo, sp.a, sp.sink, sp.n, u0, u1, kvh, split, pw, again,
                         lds_at(&kbuf[0][0]) + wv * 16 * DP);
}

// Joins the chunks of tiles that have several: W waves for a row's head, L lanes
// to a chunk's sums (four values each), so that 64 W / L chunks are read at once.
template <int KV, class T, int W, int L>
__global__ __launch_bounds__(256) void k_attn_join(KvAttnArgs g, long long unit0) {
  constexpr int N = W * 64 / L, PER = 4 / W;
  __shared__ __align__(16) float sums[W > 1 ? W : 1][W > 1 ? 4 * L : 4];
  __shared__ f32x4 stats[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const long long unit = unit0 + (long long)blockIdx.x * PER + wv / W;
  const int me = wv % W * (64 / L) + lane / L, d = 4 * (lane % L);   // this lane's chunks me, me + N, ..
  const bool there = unit < (long long)g.kv.n_rows * g.n_q;
  const int row = (int)g.by_heads((uint32_t)(there ? unit : 0)), head = there ? (int)unit - row * g.n_q : 0, D = g.kv.dim;
  KvSeq sq;
  const int s = kv_seq_of(g.kv, row, &sq);
  int n = 0;
  if (there && s >= 0) {
    const bool few = sq.rows * g.group <= g.few_rows;
    const int tile = few ? kKvFewTile : kKvManyTile;
    const int p0 = ((row - sq.first) * g.group + head_in(g, head)) & -tile;
    const int t0 = row_in(g, p0), t1 = min(row_in(g, p0 + tile - 1), sq.rows - 1);
    n = kv_splits(g, few ? kv_span<32>(g, sq, t0, t1) : kv_span<64>(g, sq, t0, t1));
  }
  if (n < 2) return;   // W > 1: the same in all of the block
  const long long step = (long long)g.kv.n_rows * g.n_q;
  // with a running reference, as the chunks themselves
  float top = -INFINITY, sum = 0.f, exact = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = me; i < n; i += N) {
    const f32x4 ml = *(const f32x4*)(g.part_ml + 4 * (unit + i * step));
    const f32x4 part = d < D ? *(const f32x4*)(g.part_o + (unit + i * step) * D + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float m = fmaxf(top, ml.x), f = top == m ? 1.f : __builtin_amdgcn_exp2f(top - m), h = ml.x == m ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
    sum = f * sum + h * ml.y;
    exact = f * exact + h * ml.z;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = scaled(v[k], f) + scaled(part[k], h);
    top = m;
  }
  float all = top;
#pragma unroll
  for (int o = L; o < 64; o <<= 1) all = fmaxf(all, __shfl_xor(all, o, 64));
  if constexpr (W > 1) {
    if (lane == 0) stats[wv].x = all;
    __syncthreads();
    all = fmaxf(fmaxf(stats[0].x, stats[1].x), fmaxf(stats[2].x, stats[3].x));
    __syncthreads();
  }
  const float f = top == all ? 1.f : __builtin_amdgcn_exp2f(top - all);
  sum *= f;
  exact *= f;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = scaled(v[k], f);
#pragma unroll
  for (int o = L; o < 64; o <<= 1) {
    sum += __shfl_xor(sum, o, 64);
    exact += __shfl_xor(exact, o, 64);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += __shfl_xor(v[k], o, 64);
  }
  if constexpr (W > 1) {
    if (lane == 0) stats[wv] = f32x4{0.f, sum, exact, 0.f};
    if (lane < L) *(f32x4*)&sums[wv][d] = v;
    __syncthreads();
    if (wv > 0) return;
    sum = exact = 0.f;
    v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sum += stats[w].y;
      exact += stats[w].z;
      if (lane < L) v += *(const f32x4*)&sums[w][d];
    }
  }
  if (lane < L && d < D) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)g.out + row * g.ldo + (long long)head * D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (T)scaled(v[i], inv);
  }
  if (lane == 0 && g.lse) g.lse[unit] = lse_of<KV>(all, exact);
}

template <int KV, class T, int W, int L>
int join_launch(const KvAttnArgs& g, hipStream_t s) {
  constexpr long long MOST = 1ll << 22, PER = 4 / W;   // blocks
  const long long units = (long long)g.kv.n_rows * g.n_q;
  for (long long at = 0; at < units; at += MOST * PER) {
    hipLaunchKernelGGL((k_attn_join<KV, T, W, L>), dim3((unsigned)((std::min(units - at, MOST * PER) + PER - 1) / PER)), dim3(256), 0, s, g, at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}
template <int KV, class T, int L>
int join_waves(const KvAttnArgs& g, hipStream_t s) {
  // four waves where a wave would take more than eight turns (48 rows of 256, 256 chunks: 46 us with one)
  return g.splits > 8 * (64 / L) ? join_launch<KV, T, 4, L>(g, s) : join_launch<KV, T, 1, L>(g, s);
}

long long slots_of(const KvAttnArgs& g, int tile) {
  return ((long long)g.kv.n_rows * g.group + (long long)(tile - 1) * g.kv.n_seqs) / tile;
}

template <int KV, int DP, class T>
int attn_launch(const KvAttnArgs& g, hipStream_t s) {
  // launches of fewer than 2^24 blocks: a grid holds fewer than 2^32 threads
  const long long each = (long long)g.kv.n_kv * g.splits;
  const long long most = std::max(1ll, ((1ll << 24) - 1) / each);
  if (g.few_rows > 0) {
    const long long slots = g.few_rows == 0x7fffffff ? slots_of(g, kKvFewTile)
                                                     : (long long)g.kv.n_seqs * kKvFewTiles;
    for (long long at = 0; at < slots; at += most) {
      const int n = (int)std::min(most, slots - at);
      hipLaunchKernelGGL((k_attn_few<KV, DP, T>), dim3((unsigned)(n * each)), dim3(256), 0, s, g, (int)at, n);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
    }
  }
  if (g.few_rows < 0x7fffffff) {
    const long long slots = slots_of(g, kKvManyTile);
    for (long long at = 0; at < slots; at += most) {
      const int n = (int)std::min(most, slots - at);
      hipLaunchKernelGGL((k_attn_many<KV, DP, T>), dim3((unsigned)(n * each)), dim3(256), 0, s, g, (int)at, n);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
    }
  }
  if (g.splits == 1) return 0;
  return g.kv.dim <= 64 ? join_waves<KV, T, 16>(g, s) : g.kv.dim <= 128 ? join_waves<KV, T, 32>(g, s) : join_waves<KV, T, 64>(g, s);
}
template <int KV, class T>
int attn_dim(const KvAttnArgs& g, hipStream_t s) {
  if (g.kv.dim <= 64) return attn_launch<KV, 64, T>(g, s);
  if (g.kv.dim <= 128) return attn_launch<KV, 128, T>(g, s);
  return attn_launch<KV, 256, T>(g, s);
}
template <int KV>
int attn_type(int elem, const KvAttnArgs& g, hipStream_t s) {
  switch (elem) {
    case ELEM_F32: return attn_dim<KV, float>(g, s);
    case ELEM_F16: return attn_dim<KV, _Float16>(g, s);
    case ELEM_BF16: return attn_dim<KV, __bf16>(g, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace

// The chunk length is taken from estimates of a call's time, in us, over the
// numbers of chunks; lengths are taken to be spread between 0 and max_len.
// k_attn_few: a block starts and ends in 5 us and takes 128 keys in 1.2, or as long as
// 5 TB/s need for what all resident blocks read; a join takes 3 and 0.1 a chunk.
// k_attn_many: whole rounds of the CUs; a block's start and end cost about 200
// keys, a chunk's sums are written and read once more.
// Measured at the two sides of the choice, us, on three sets of inputs in turn,
// which no cache holds together: 16 times 6 drafts to 4096 positions, 16 heads of 128 on 8, the estimate's
// 7 chunks 50, 1 62, 2 70, 3 52, 5 47.5, 8 48; 61 tokens to 8192, its 8 229, 2 257, 4 233,
// 12 229; 3 tokens to 131072, 8-bit heads of 256, its 18 142, 16 147, 24 210, 64 151,
// 256 174; 2048 rows at 32768, 4 heads of 256 on 1, its 4 329, 3 431, 5 528, 8 356;
// windowed f32 turns, its 2 67.5, 1 80, 3 95.
KvAttnPlan kv_attn_plan(int n_seqs, int n_rows, int max_rows, int max_len, int n_kv, int group, int dim, int window, int sinks,
                        int key_bytes) {
  KvAttnPlan p{};
  constexpr int FEW = kKvFewTiles * kKvFewTile;
  const bool few = (long long)max_rows * group <= FEW;
  // Long ones: k_attn_many alone, a launch less; what is short among them it can do
  // too. A prompt beside single tokens at up to 8192 positions, us with k_attn_many
  // alone / both, 4 heads of 256 on 1 and 32 of 128 on 8: 4096 rows and 31 tokens
  // 245 / 265 and 386 / 391, 8192 and 31 465 / 522 and 901 / 960; below the border 256 and 31
  // 77 / 69 and 176 / 163. Near it neither is always the better: 2048 and 31 150 / 158 and
  // 248 / 259, 300 and 1 28 / 40 but 58 / 41.
  p.few_rows = few ? 0x7fffffff : (long long)n_rows * group >= 512ll * n_seqs ? 0 : FEW;
  const int tile = few ? kKvFewTile : kKvManyTile;
  long long most = max_len;   // keys that a tile's rows see at most
  if (window > 0) most = std::min(most, (long long)window + tile) + ((long long)std::min(sinks, max_len) + 63) / 64 * 64;
  const long long packed = (long long)n_rows * group, of_seq = (packed + n_seqs - 1) / n_seqs;
  const double tiles = (double)n_seqs * (double)((of_seq + tile - 1) / tile) * n_kv;
  const double share = window > 0 ? 1.0 : 0.5 + 0.5 / n_seqs;
  double best = 1e300;
  long long chunk = most;
  for (long long c = 1; c <= 256 && (c - 1) * kKvChunk < most; ++c) {
    const long long len = ((most + c - 1) / c + kKvChunk - 1) / kKvChunk * kKvChunk;
    double cost;
    if (few) {
      const double blocks = tiles * (most * share / len + (n_seqs > 1 ? 0.5 : 0.0));
      const double rounds = std::max(1.0, blocks / 256 + (n_seqs > 1 ? 0.4 : 0.0));
      cost = rounds * (5.0 + len / 128 * std::max(1.2, 128.0 * key_bytes / 5e6 * std::min(blocks, 256.0))) + (c > 1 ? 3.0 + 0.1 * c : 0.0);
    } else {
      if (c > 64) break;
      const double real = std::max(1.0, (double)((packed + tile - 1) / tile * n_kv));
      cost = std::ceil(real * c / 256) * (len + 200.0) * dim / 256 +
             (c > 1 ? 100.0 + 0.06 * c * n_rows * group * n_kv * dim / 32768 : 0.0);
    }
    if (cost < best) {
      best = cost;
      chunk = len;
    }
  }
  p.chunk = (int)std::min(chunk, (most + kKvChunk - 1) / kKvChunk * kKvChunk);
  p.splits = (int)((most + p.chunk - 1) / p.chunk);
  return p;
}

int launch_kv_attention(int kv_type, int elem, const KvAttnArgs& g, void* stream) {
  switch (kv_type) {
    case KV_BF16: return attn_type<KV_BF16>(elem, g, (hipStream_t)stream);
    case KV_F16: return attn_dim<KV_F16, _Float16>(g, (hipStream_t)stream);
    case KV_E4M3: return attn_type<KV_E4M3>(elem, g, (hipStream_t)stream);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
