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
__device__ __forceinline__ Span kv_span(const KvAttnArgs& g, const KvSeq& sq, int row_first, int row_last) {
  Span s{};
  const int before = sq.len - sq.rows;
  const int hi = min(before + row_last + 1, g.kv.places);
  if (hi <= 0) return s;
  s.lo = g.window > 0 ? max(0, before + row_first - g.window + 1) : 0;
  s.sink = g.window > 0 ? min(min(g.sinks, s.lo), hi) : 0;
  s.a = (s.sink + 31) / 32 * 32;
  s.n = s.a + max(0, hi - s.lo);
  return s;
}
__device__ __forceinline__ int kv_splits(const KvAttnArgs& g, const Span& s) { return max(1, (s.n + g.chunk - 1) / g.chunk); }

// The slots of a sequence's tiles: consecutive from floor(first row group / tile) + s
// on, enough for tiles of whole sequences, so that a slot's sequence is found
// by search and no list of tiles is made.
__device__ __forceinline__ long long tile_slot(const KvAttnArgs& g, int s, int tile) {
  return (long long)min(max(g.kv.row_start[s], 0), g.kv.n_rows) * g.group / tile + s;
}

// ln of a sum of weights relative to m (log2 units).
template <int KV>
__device__ __forceinline__ float lse_of(float m, float sum) {
  return sum == 0.f ? -INFINITY : (m - kShift<KV> + __builtin_amdgcn_logf(sum)) * kLn2;
}

// A sum times a factor that is not 0 but may have become it: an infinity stays.
__device__ __forceinline__ float scaled(float x, float f) { return fabsf(x) == INFINITY ? x : x * f; }

// Whether a 16-bit value is an infinity or a NaN.
template <int KV>
__device__ __forceinline__ bool odd_value(uint32_t h) {
  constexpr uint32_t M = KV == KV_F16 ? 0x7c00u : 0x7f80u;
  return (h & M) == M;
}

// ---------------------------------------------------------------------------
// Few rows: a block takes 16 packed rows of a K/V head and a chunk of keys, its
// waves 32 keys at a time in turn. K and V go from memory to registers, K in
// operand order as it lies, V in rows (16 lanes share one) and transposed by
// byte permutes: no LDS, no barrier in the loop; the next step's K is asked for
// when this one's is used up, V likewise.
// ---------------------------------------------------------------------------
template <int KV, int DP, class T>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_attn_few(KvAttnArgs g, int slot0) {
  constexpr int NP = kParts<KV, T>, KC = DP / 32, VD = DP / 16, OP = DP + 4;
  constexpr int ES = KV == KV_E4M3 ? 1 : 2;                 // bytes of an element in the pages
  constexpr int KW = 2 * ES, VW = VD * ES / 4;              // dwords a lane loads of a K chunk, of a V row
  __shared__ __align__(16) float o_all[4][kKvFewTile][OP];
  __shared__ float m_all[4][kKvFewTile], l_all[4][kKvFewTile], e_all[4][kKvFewTile];
  __shared__ __align__(16) long long key_off[4][32];        // where a step's rows lie, -1: nowhere
  __shared__ __align__(16) float k_sc[4][32], v_sc[4][32];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, quad = lane >> 4, D = g.kv.dim;
  const int split = blockIdx.x % g.splits, hs = blockIdx.x / g.splits;
  const int kvh = hs % g.kv.n_kv, slot = slot0 + hs / g.kv.n_kv;
  const int s = last_at_most(g.kv.n_seqs, [&](int i) { return tile_slot(g, i, kKvFewTile) <= slot; });
  if (s < 0) return;
  const KvSeq sq = kv_seq(g.kv, s);
  const long long tile_l = slot - tile_slot(g, s, kKvFewTile);
  const int packed = sq.rows * g.group;
  if (tile_l < 0 || tile_l * kKvFewTile >= packed || packed > g.few_rows) return;
  const int p0 = (int)tile_l * kKvFewTile;
  const Span sp = kv_span(g, sq, p0 / g.group, min((p0 + kKvFewTile - 1) / g.group, sq.rows - 1));
  const int u0 = split * g.chunk, u1 = min(sp.n, u0 + g.chunk);
  if (split > 0 && u0 >= sp.n) return;
  const bool joined = kv_splits(g, sp) > 1;

  // this lane's packed row: its query as operand columns, its position
  const int p = p0 + c16, row = sq.first + p / g.group, head = kvh * g.group + p % g.group;
  const int pos = p < packed ? sq.len - sq.rows + p / g.group : -1;
  u32x4 qb[NP][KC];
  {
    const T* q = (const T*)g.q + (p < packed ? row * g.ldq + (long long)head * D : 0);
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = 32 * c + 8 * quad;
      float f[8] = {};
      if (p < packed && d < D) {
        if (g.q_vec) {
          constexpr int V = 16 / sizeof(T);
          typedef T vec_t __attribute__((ext_vector_type(V)));
#pragma unroll
          for (int i = 0; i < 8; i += V) {
            const vec_t t = *(const vec_t*)(q + d + i);
#pragma unroll
            for (int k = 0; k < V; ++k) f[i + k] = (float)t[k];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = (float)q[d + i];
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

  f32x4 o[VD];
#pragma unroll
  for (int t = 0; t < VD; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f, le = 0.f;   // le: of the weights before they are rounded, for lse
  typedef uint32_t kw_t __attribute__((ext_vector_type(KW)));
  typedef uint32_t vw_t __attribute__((ext_vector_type(VW > 4 ? 4 : VW)));
  constexpr int VN = VW > 4 ? VW / 4 : 1;
  kw_t kr[2][KC];
  vw_t vr[8][VN];
  long long voff[8];

  // The places of a step's keys, one a lane, into LDS.
  auto places = [&](int u) __attribute__((always_inline)) {
    if (lane < 32) {
      const int x = u + lane, key = x < sp.a ? x : sp.lo + x - sp.a;
      KvPlace at{};
      const bool ok = x < u1 && (x >= sp.a || x < sp.sink) && kv_place(g.kv, s, key, &at);
      key_off[wv][lane] = ok ? kv_offset(g.kv, at, kvh) : -1;
      if constexpr (KV == KV_E4M3) {
        k_sc[wv][lane] = ok ? g.kv.k_scale[kv_scale_at(g.kv, at, kvh)] : 0.f;
        v_sc[wv][lane] = ok ? g.kv.v_scale[kv_scale_at(g.kv, at, kvh)] : 0.f;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long off = max(key_off[wv][16 * h + c16], 0ll);
      const uint8_t* r = (const uint8_t*)g.kv.k + off * ES;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int d = 32 * c + 8 * quad;
        kr[h][c] = *(const kw_t*)(r + (d < D ? d : 0) * ES);   // past D the query is 0
      }
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
    const int d = VD * c16;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      voff[j] = key_off[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
      const uint8_t* r = (const uint8_t*)g.kv.v + (max(voff[j], 0ll) + (d < D ? d : 0)) * ES;
#pragma unroll
      for (int n = 0; n < VN; ++n) vr[j][n] = ((const vw_t*)r)[n];
    }
  };

  // All of this wave's keys. `careful`: infinities and NaN of V reach the rows
  // that see their keys and no others.
  auto pass = [&](auto careful) __attribute__((always_inline)) {
  int u = u0 + 32 * wv;
  float ks[8], vs[8];
  if (u < u1) {
    places(u);
    load_k();
    if constexpr (!careful) load_v();
  }
  for (; u < u1; u += 128) {
    if constexpr (KV == KV_E4M3) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ks[j] = k_sc[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
        vs[j] = v_sc[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
      }
    }
    bool here[8], miss = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (careful) voff[j] = key_off[wv][4 * quad + (j & 3) + 16 * (j >> 2)];
      here[j] = voff[j] >= 0;
      miss |= !here[j];
    }
    // S^T: 32 keys x 16 packed rows
    f32x4 sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        u32x4 ka;
        if constexpr (KV == KV_E4M3) {
          typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
          const bf16x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kr[h][c][0], 1.f, false),
                       a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kr[h][c][0], 1.f, true),
                       a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kr[h][c][1], 1.f, false),
                       a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kr[h][c][1], 1.f, true);
          ka = u32x4{__builtin_bit_cast(uint32_t, a0), __builtin_bit_cast(uint32_t, a1), __builtin_bit_cast(uint32_t, a2),
                     __builtin_bit_cast(uint32_t, a3)};
        } else {
          ka = kr[h][c];
        }
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) sc[h] = mfma16<KV>(ka, qb[k][c], sc[h]);
      }
    }
    const int next = u + 128;
    if (next < u1) {
      places(next);
      load_k();
    }
    // scores in log2 units; what the row does not see is -inf
    const int key0 = u < sp.a ? u : sp.lo + u - sp.a;
    float x[8], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = key0 + 4 * quad + (j & 3) + 16 * (j >> 2);
      const bool sees = key <= pos && (g.window == 0 || key > pos - g.window || key < g.sinks);
      float t = sc[j >> 2][j & 3] * g.scale2;
      if constexpr (KV == KV_E4M3) t *= ks[j];
      x[j] = here[j] && sees ? t : -INFINITY;
      here[j] = here[j] && sees;
      mx = fmaxf(mx, x[j]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    float f = 1.f;
    if (__ballot(mx > m + kSlack)) {
      const float mn = mx > m + kSlack ? mx : m;
      f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
      le *= f;
      if constexpr (!careful) {
#pragma unroll
        for (int t = 0; t < VD; ++t) o[t] *= f;
      }
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
        w0 = here[2 * i] ? w0 * vs[2 * i] : 0.f;
        w1 = here[2 * i + 1] ? w1 * vs[2 * i + 1] : 0.f;
      }
      if constexpr (NP > 1 || KV == KV_E4M3) split2<KV, NP>(w0, w1, w);
#pragma unroll
      for (int k = 0; k < NP; ++k) pb[k][i] = w[k];
    }
    // V of keys that are not there counts as 0: what lies there may be a NaN
    if (!careful && __ballot(miss)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int n = 0; n < VN; ++n) vr[j][n] = voff[j] >= 0 ? vr[j][n] : (vw_t)0;
    }
    // 16-bit rows of V: dword i of key j holds values 2i and 2i + 1
    auto v_word = [&](int j, int i) __attribute__((always_inline)) -> uint32_t {
      if constexpr (KV == KV_E4M3) {
        const uint32_t w = vr[j][(i / 2) / 4][(i / 2) % 4];
        return i % 2 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))
                     : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
      } else {
        return vr[j][i / 4][i % 4];
      }
    };
    if constexpr (careful) {
      // sums in LDS, one value of a head at a time: the finite values as ever, then
      // the infinities of either sign among the keys that the row sees (a NaN is both)
      constexpr uint32_t ONE = KV == KV_F16 ? 0x3c00u : 0x3f80u, MANT = KV == KV_F16 ? 0x3ffu : 0x7fu;
      u32x4 seen;
#pragma unroll
      for (int i = 0; i < 4; ++i) seen[i] = (here[2 * i] ? ONE : 0u) | (here[2 * i + 1] ? ONE << 16 : 0u);
#pragma unroll 1
      for (int t = 0; t < VD; ++t) {
        const int d = VD * c16 + t;
        u32x4 clean, up, down;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t cl[2], pu[2], pd[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t h = 0;
            if (voff[2 * i + e] >= 0 && d < D) {
              const uint8_t* r = (const uint8_t*)g.kv.v + (voff[2 * i + e] + d) * ES;
              if constexpr (KV == KV_E4M3)
                h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)*r, 1.f, false)) & 0xffffu;
              else
                h = *(const uint16_t*)r;
            }
            const bool is_odd = odd_value<KV>(h), nan = is_odd && (h & MANT);
            cl[e] = is_odd ? 0u : h;
            pu[e] = is_odd && (nan || !(h & 0x8000u)) ? ONE : 0u;
            pd[e] = is_odd && (nan || (h & 0x8000u)) ? ONE : 0u;
          }
          clean[i] = cl[0] | (cl[1] << 16);
          up[i] = pu[0] | (pu[1] << 16);
          down[i] = pd[0] | (pd[1] << 16);
        }
        float* sum = &o_all[wv][c16][4 * VD * quad + t];
        f32x4 c;
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = scaled(sum[VD * i], f);
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) c = mfma16<KV>(clean, pb[k], c);
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 nu = mfma16<KV>(up, seen, zero), nd = mfma16<KV>(down, seen, zero);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (nu[i] > 0.f) c[i] += INFINITY;
          if (nd[i] > 0.f) c[i] -= INFINITY;
          sum[VD * i] = c[i];
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < VD; t += 2) {
        u32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w0 = v_word(2 * i, t / 2), w1 = v_word(2 * i + 1, t / 2);
          lo[i] = lower2(w0, w1);
          hi[i] = upper2(w0, w1);
        }
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) {
          o[t] = mfma16<KV>(lo, pb[k], o[t]);
          o[t + 1] = mfma16<KV>(hi, pb[k], o[t + 1]);
        }
      }
    }
    if (!careful && next < u1) load_v();
  }
  };
  // A weight of 0, or a part of one, times an infinity or a NaN leaves a NaN, so
  // whatever needs care shows in O, and the main loop need not look at V.
  pass(std::false_type{});
  bool again;
  {
    float z = 0.f;
#pragma unroll
    for (int t = 0; t < VD; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) z = fmaf(o[t][i], 0.f, z);
    again = __ballot(z != 0.f) != 0;   // 0 times an infinity or a NaN
  }
  if (again) {
    for (int e = lane; e < kKvFewTile * OP; e += 64) (&o_all[wv][0][0])[e] = 0.f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    m = -INFINITY;
    l = le = 0.f;
    pass(std::true_type{});
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
    if (again) {
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
    const long long orow = sq.first + pr / g.group;
    const int oh = kvh * g.group + pr % g.group;
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

// Joins the chunks of tiles that have several: one wave for a row's head.
template <int KV, class T>
__global__ __launch_bounds__(256) void k_attn_join(KvAttnArgs g, long long unit0) {
  const int lane = threadIdx.x & 63;
  const long long unit = unit0 + (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= (long long)g.kv.n_rows * g.n_q) return;
  const int row = (int)(unit / g.n_q), head = (int)(unit % g.n_q), D = g.kv.dim;
  const int s = kv_seq_of(g.kv, row);
  if (s < 0) return;
  const KvSeq sq = kv_seq(g.kv, s);
  const int tile_rows = kKvFewTile;
  const int p0 = ((row - sq.first) * g.group + head % g.group) / tile_rows * tile_rows;
  const Span sp = kv_span(g, sq, p0 / g.group, min((p0 + tile_rows - 1) / g.group, sq.rows - 1));
  const int n = kv_splits(g, sp);
  if (n < 2) return;
  const long long step = (long long)g.kv.n_rows * g.n_q;
  float top = -INFINITY;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, g.part_ml[4 * (unit + i * step)]);
  top = wave_max(top);
  float sum = 0.f, exact = 0.f;
  for (int i = lane; i < n; i += 64) {
    const f32x4 ml = *(const f32x4*)(g.part_ml + 4 * (unit + i * step));
    const float f = ml.x == top ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
    sum += f * ml.y;
    exact += f * ml.z;
  }
  sum = wave_sum(sum);
  exact = wave_sum(exact);
  const int d = 4 * lane;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (d < D) {
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float m = g.part_ml[4 * (unit + i * step)];
      const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
      const f32x4 part = *(const f32x4*)(g.part_o + (unit + i * step) * D + d);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += scaled(part[k], f);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)g.out + row * g.ldo + (long long)head * D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (T)(v[i] * inv);
  }
  if (lane == 0 && g.lse) g.lse[unit] = lse_of<KV>(top, exact);
}

template <int KV, int DP, class T>
int attn_launch(const KvAttnArgs& g, hipStream_t s) {
  // launches of fewer than 2^24 blocks: a grid holds fewer than 2^32 threads
  const long long slots = (long long)g.kv.n_rows * g.group / kKvFewTile + g.kv.n_seqs;
  const long long each = (long long)g.kv.n_kv * g.splits;
  const long long most = std::max(1ll, ((1ll << 24) - 1) / each);
  for (long long at = 0; at < slots; at += most) {
    hipLaunchKernelGGL((k_attn_few<KV, DP, T>), dim3((unsigned)(std::min(most, slots - at) * each)), dim3(256), 0, s, g, (int)at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (g.splits == 1) return 0;
  const long long units = (long long)g.kv.n_rows * g.n_q;
  for (long long at = 0; at < units; at += 1ll << 25) {
    hipLaunchKernelGGL((k_attn_join<KV, T>), dim3((unsigned)((std::min(units - at, 1ll << 25) + 3) / 4)), dim3(256), 0, s, g, at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
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

KvAttnPlan kv_attn_plan(int n_seqs, int n_rows, int max_rows, int max_len, int n_kv, int group, int dim, int window, int sinks) {
  KvAttnPlan p{};
  p.few_rows = 0x7fffffff;
  long long most = max_len;   // keys that a tile's rows see at most
  if (window > 0) most = std::min(most, (long long)window + kKvFewTile) + ((long long)std::min(sinks, max_len) + 31) / 32 * 32;
  most = std::max(most, 1ll);
  const long long tiles = ((long long)n_rows * group / kKvFewTile + n_seqs) * n_kv;
  long long chunk = (most * tiles / 4096 + kKvChunk) / kKvChunk * kKvChunk;
  chunk = std::max(chunk, most <= 2048 ? 128ll : 512ll);
  p.chunk = (int)std::min(chunk, (most + kKvChunk - 1) / kKvChunk * kKvChunk);
  p.splits = (int)((most + p.chunk - 1) / p.chunk);
  return p;
}

int launch_kv_attention(int kv_type, int elem, const KvAttnArgs& g, int max_rows, void* stream) {
  switch (kv_type) {
    case KV_BF16: return attn_type<KV_BF16>(elem, g, (hipStream_t)stream);
    case KV_F16: return attn_dim<KV_F16, _Float16>(g, (hipStream_t)stream);
    case KV_E4M3: return attn_type<KV_E4M3>(elem, g, (hipStream_t)stream);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
