// gg_mxfp4.hip -- MXFP4 matrices on gfx950: quantisation, expansion, and
// products y = x W^T with W in MXFP4 and x in f32 / f16 / bf16 or MXFP4.
// The formats and layouts are described at Mx4Layout and mx_parts
// (gg_internal.h).
#include "gg_device.h"

#include <algorithm>

namespace gg {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
constexpr int kFp4 = 4;   // operand format of the MX matrix instructions
template <class T>
constexpr int kElem = __is_same(T, float) ? ELEM_F32 : __is_same(T, _Float16) ? ELEM_F16 : ELEM_BF16;

// Elements [c, c + E) of a row of k elements, zeros past its end.
template <class T, int E, bool VEC, bool NT = false>
__device__ __forceinline__ void load_row(const T* row, int64_t c, int64_t k, float (&v)[E]) {
  typedef T vec_t __attribute__((ext_vector_type(E)));
  if (VEC && c + E <= k) {
    const vec_t t = NT ? __builtin_nontemporal_load((const vec_t*)(row + c)) : *(const vec_t*)(row + c);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = c + i < k ? (float)row[c + i] : 0.f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void load4(const T* row, int64_t c, int64_t k, float (&v)[4]) { load_row<T, 4, VEC>(row, c, k, v); }

// ---------------------------------------------------------------------------
// Quantisation. A block takes 32 rows x 256 k (one group of scale dwords): a
// wave reads 16 bytes a lane, 256 consecutive elements of one f32 row or of two
// 16-bit ones at a time, 8 or 4 lanes to a 32-block; the codes go through LDS
// into operand order, so that both the reads and the 1 KB tiles written are
// whole lines.
// Scale byte: the exponent field of the block's largest magnitude less 2
// (floor(log2) - 2), at least 0; conversion to nearest, ties to even, values
// above 6 to 6. Bound by memory: reads the input once, writes 17/32 byte an
// element (262144 x 1152 bf16, 764 MB: 141 us, 5.4 TB/s; 187 x 6912 f32 3.8 us,
// three times an empty kernel).
// ---------------------------------------------------------------------------
template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_mx4_quantize(const T* __restrict__ src, int64_t rows, int64_t k, int64_t ld,
                                                      uint8_t* __restrict__ dst, Mx4Layout L, int64_t r0) {
  constexpr int E = 16 / sizeof(T), LB = 32 / E, RW = E / 4;   // elements a lane, lanes a block, rows a wave at a time
  __shared__ __align__(16) uint8_t codes[256][16];   // [4 tiles x 64 lanes][16 bytes]
  __shared__ __align__(4) uint8_t scales[256];       // [64 lanes][4 tiles]
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = r0 + blockIdx.x;
  const int g = blockIdx.y;
  const int ln = lane % (64 / RW);
  const int64_t c = (int64_t)g * 256 + E * ln;
  const int kb = ln / LB, t = kb >> 1, b = kb & 1;   // 32-block, its tile and half
  float v[8 / RW][E];
  if constexpr (VEC || sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8 / RW; ++i) {
      const int64_t r = R * 32 + wv * 8 + i * RW + lane / (64 / RW);
      load_row<T, E, VEC, VEC>(src + min(r, rows - 1) * ld, c, r < rows ? k : 0, v[i]);
    }
  } else {
    // 16-bit rows at odd addresses: an element a lane, whole lines all the
    // same, and to the lanes that take them through LDS (20000 x 1153 bf16 33
    // -> 25 us; f32 rows, four loads a lane, take 25 as they are and 40 so)
    __shared__ __align__(16) T rowbuf[4][8][256];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = R * 32 + wv * 8 + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t e = (int64_t)g * 256 + 64 * j + lane;
        rowbuf[wv][i][64 * j + lane] = r < rows && e < k ? src[r * ld + e] : (T)0.f;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < 8 / RW; ++i) {
      typedef T vec_t __attribute__((ext_vector_type(E)));
      const vec_t t = *(const vec_t*)&rowbuf[wv][i * RW + lane / (64 / RW)][E * ln];
#pragma unroll
      for (int j = 0; j < E; ++j) v[i][j] = (float)t[j];
    }
  }
#pragma unroll
  for (int i = 0; i < 8 / RW; ++i) {
    const int row = wv * 8 + i * RW + lane / (64 / RW);
    // the magnitudes' bits order as the magnitudes do, Inf and NaN on top
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) a = max(a, __float_as_uint(v[i][j]) & 0x7fffffffu);
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xf, 0xf, false));
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xf, 0xf, false));
    if (LB == 8) a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x141, 0xf, 0xf, false));
    const int ex = (int)(a >> 23);
    const int byte = ex == 255 ? 255 : max(ex - 2, 0);
    const float scale = __uint_as_float(byte ? (uint32_t)byte << 23 : 0x00400000u);   // byte 0: 2^-127
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][0], v[i][1], scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][2], v[i][3], scale, 1);
    if constexpr (E == 8) {
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][4], v[i][5], scale, 2);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][6], v[i][7], scale, 3);
    }
    if (byte == 255) q = 0;   // Inf or NaN in the block: its scale says NaN
    const int l = 32 * b + row;
    if constexpr (E == 8) *(uint32_t*)&codes[t * 64 + l][4 * (ln % LB)] = q;
    else *(uint16_t*)&codes[t * 64 + l][2 * (ln % LB)] = (uint16_t)q;
    if (ln % LB == 0) scales[4 * l + t] = (uint8_t)byte;
  }
  __syncthreads();
  if (g * 4 + wv < L.kt)
    *(u32x4*)(dst + ((size_t)R * L.kt + g * 4 + wv) * 1024 + 16 * lane) = *(const u32x4*)codes[wv * 64 + lane];
  if (wv == 0)
    *(uint32_t*)(dst + L.codes() + ((size_t)R * L.ks + g) * 256 + 4 * lane) = *(const uint32_t*)(scales + 4 * lane);
}

// ---------------------------------------------------------------------------
// Expansion to f32, the same tile the other way: each value is its 4-bit
// element times 2^(byte - 127), NaN where the byte is 255. Bound by the f32
// write (262144 x 1152, 1.37 GB: 235 us, 5.8 TB/s).
// ---------------------------------------------------------------------------
template <bool VEC>
__global__ __launch_bounds__(256) void k_mx4_dequant(const uint8_t* __restrict__ src, float* __restrict__ out,
                                                     int64_t rows, int64_t k, int64_t ld, Mx4Layout L, int64_t r0) {
  __shared__ __align__(16) uint16_t codes[256][8];
  __shared__ __align__(4) uint8_t scales[256];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = r0 + blockIdx.x;
  const int g = blockIdx.y;
  if (g * 4 + wv < L.kt)
    *(u32x4*)codes[wv * 64 + lane] = *(const u32x4*)(src + ((size_t)R * L.kt + g * 4 + wv) * 1024 + 16 * lane);
  if (wv == 0)
    *(uint32_t*)(scales + 4 * lane) = *(const uint32_t*)(src + L.codes() + ((size_t)R * L.ks + g) * 256 + 4 * lane);
  __syncthreads();
  const int64_t c = (int64_t)g * 256 + 4 * lane;
  const int kb = lane >> 3, t = kb >> 1, b = kb & 1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = wv * 8 + i;
    const int64_t r = R * 32 + row;
    if (r >= rows) continue;
    const int l = 32 * b + row;
    const uint32_t q = codes[t * 64 + l][lane & 7];
    const int byte = scales[4 * l + t];
    // the elements on their own, then the power of two in f32 (2^-127 and
    // products below 2^-126 are denormal and exact)
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    const float v[4] = {lo[0], lo[1], hi[0], hi[1]};
    f32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = byte == 255 ? NAN : ldexpf(v[j], byte - 127);
    float* d = out + r * ld;
    if constexpr (VEC) {
      if (c + 4 <= k) {
        __builtin_nontemporal_store(o, (f32x4*)(d + c));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < k) d[c + j] = o[j];
      }
    } else {
      // rows at odd addresses: an element a lane
      __shared__ __align__(16) float rowbuf[4][256];
      *(f32x4*)&rowbuf[wv][4 * lane] = o;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t e = (int64_t)g * 256 + 64 * j + lane;
        const float t = rowbuf[wv][64 * j + lane];
        if (e < k) d[e] = t;   // through the cache, which makes whole lines of them
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// ---------------------------------------------------------------------------
// Activations in parts (mx_parts): a part of a value is the upper 16 bits of
// what is left of it in f32, a bf16 towards zero, so that no part rounds and
// none overflows: 8 significant bits each, 24 in three. A subtraction of the
// upper bits is exact. An infinity leaves NaN behind it; bf16 x, which has one
// part, turns into NaN here.
// ---------------------------------------------------------------------------
__device__ __forceinline__ u32x4 take_part(float (&u)[8]) {
  u32x4 z;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a = __float_as_uint(u[2 * j]), b = __float_as_uint(u[2 * j + 1]);
    z[j] = __builtin_amdgcn_perm(b, a, 0x07060302);
    u[2 * j] -= __uint_as_float(a & 0xffff0000u);
    u[2 * j + 1] -= __uint_as_float(b & 0xffff0000u);
  }
  return z;
}
template <class T>
__device__ __forceinline__ void inf_to_nan(float (&u)[8]) {
  if constexpr (__is_same(T, __bf16)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = __builtin_fabsf(u[j]) == INFINITY ? NAN : u[j];
  }
}

// A wave takes 32 rows x 64 k, a thread one 32-block of them. The rows come in
// whole lines, four elements a lane (one where their addresses are odd), and
// change lanes in LDS; a pitch of 68 floats puts the 16 lanes of a read on
// different banks. Bound by memory for long x (reads 4 or 2 bytes, writes 2 a
// part and element; 4000 x 8192 bf16, 131 MB: 23 us, 5.7 TB/s), by its latency for
// short (2048 x 1152 f32, 24 MB: 8 us).
template <class T, bool VEC>
__global__ __launch_bounds__(64) void k_mx_split(const T* __restrict__ src, int64_t rows, int64_t k, int64_t ld,
                                                 uint8_t* __restrict__ dst, Mx4Layout L) {
  constexpr int PITCH = 68, P = mx_parts(kElem<T>);
  __shared__ __align__(16) float xs[32 * PITCH];
  const int lane = threadIdx.x;
  const int64_t R = blockIdx.x;
  const int t = blockIdx.y;
  if constexpr (VEC) {
    float v[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = R * 32 + 4 * i + (lane >> 4);
      load4<T, true>(src + min(r, rows - 1) * ld, (int64_t)t * 64 + 4 * (lane & 15), r < rows ? k : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *(f32x4*)(xs + (4 * i + (lane >> 4)) * PITCH + 4 * (lane & 15)) = f32x4{v[i][0], v[i][1], v[i][2], v[i][3]};
  } else {
    const int64_t e = (int64_t)t * 64 + lane;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int64_t r = R * 32 + i;
      v[i] = r < rows && e < k ? (float)src[r * ld + e] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) xs[i * PITCH + lane] = v[i];
  }
  __syncthreads();
  const float* mine = xs + (lane & 31) * PITCH + 32 * (lane >> 5);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const f32x4 lo = *(const f32x4*)(mine + 8 * s), hi = *(const f32x4*)(mine + 8 * s + 4);
    float u[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    inf_to_nan<T>(u);
#pragma unroll
    for (int p = 0; p < P; ++p)
      *(u32x4*)(dst + (((size_t)t * P + p) * L.rt + R) * kMxPartBytes + 1024 * s + 16 * lane) = take_part(u);
  }
}

// Eight consecutive 4-bit weights in bf16: element times the power of two, exactly (bf16 holds what is
// denormal there too, and the matrix instruction takes it), NaN where the scale is the one of byte 255.
__device__ __forceinline__ bf16x8 expand8(uint32_t q, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1),
             c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The factor of a scale byte as the conversion reads it, from its exponent field: 0 is 2^-127 there.
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }

template <class T>
__device__ __forceinline__ void store_y(void* y, int64_t i, float v) { ((T*)y)[i] = (T)v; }
__device__ __forceinline__ void store_elem(int elem, void* y, int64_t i, float v) {
  if (elem == ELEM_F32) store_y<float>(y, i, v);
  else if (elem == ELEM_F16) store_y<_Float16>(y, i, v);
  else store_y<__bf16>(y, i, v);
}

// A wave's 32 rows x F results from LDS (row pitch P floats) to y: 16 bytes a
// lane where `vec` (rows of y 16-byte aligned) and all of them exist, else an
// element a lane; either way the lanes go along the rows.
template <class T, int F, int P>
__device__ __forceinline__ void store_tile_t(T* y, int64_t ldy, int64_t row0, int64_t f0, int64_t m, int64_t n, int vec,
                                             const float* tile, int lane) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  if (vec && f0 + F <= n) {
#pragma unroll
    for (int i = 0; i < 32 * F / (64 * V); ++i) {
      const int c = (i * 64 + lane) * V, r = c / F, f = c % F;
      vec_t o;
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const f32x4 t = *(const f32x4*)(tile + r * P + f + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * q + e] = (T)t[e];
      }
      if (row0 + r < m) *(vec_t*)(y + (row0 + r) * ldy + f0 + f) = o;
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < 32 * F / 64; ++i) {
      const int c = i * 64 + lane, r = c / F, f = c % F;
      if (row0 + r < m && f0 + f < n) y[(row0 + r) * ldy + f0 + f] = (T)tile[r * P + f];
    }
  }
}
template <int F, int P>
__device__ __forceinline__ void store_tile(int elem, void* y, int64_t ldy, int64_t row0, int64_t f0, int64_t m, int64_t n,
                                           int vec, const float* tile, int lane) {
  if (elem == ELEM_F32) store_tile_t<float, F, P>((float*)y, ldy, row0, f0, m, n, vec, tile, lane);
  else if (elem == ELEM_F16) store_tile_t<_Float16, F, P>((_Float16*)y, ldy, row0, f0, m, n, vec, tile, lane);
  else store_tile_t<__bf16, F, P>((__bf16*)y, ldy, row0, f0, m, n, vec, tile, lane);
}

// ---------------------------------------------------------------------------
// Few rows: m x parts columns in NC tiles of the 16 x 16 x 32 bf16 matrix
// instruction, column r parts + p holding part p of row r, so that four of them
// multiply 16 weight rows x 128 k by 16 columns; the weights are expanded to
// bf16 on the way, and the sum over the parts is taken once, at the end, in
// f32. One block a CU makes the
// parts in its LDS (one launch, no workspace) and goes over its share of the
// weights, which travel from memory to registers, kGemvAhead KB ahead in each
// wave. A wave takes 16 weight rows; `kw` waves of a block share their k.
// Bound by the read of the weights (17/32 byte each): 262144 x 1152 f32 28 to 30 us,
// 5.4 to 5.8 TB/s (2 us more with the addresses of a step computed from the row and
// k indices each time; 12 KB ahead are no longer kept in registers: 88 us). A small product by its chain of x,
// parts, weights, sums: 1 row, 1536 x 1152 4.8 us and 1152 x 6912 6.2 us, 7 rows of
// 13824 x 1152 6.9 us, an empty kernel 1.3.
// ---------------------------------------------------------------------------
constexpr int kGemvAhead = 8;

template <class T, int NC>
__global__ __launch_bounds__(64 * kMxGemvWaves) void k_mx4_gemv(Mx4LinearArgs a, int kw) {
  constexpr int RP = 16 * NC + 1;
  extern __shared__ f32x4 gemv_lds[];
  float* red = (float*)gemv_lds;                                       // the waves' sums
  uint8_t* rec = (uint8_t*)gemv_lds + mx_gemv_sums(NC);                // the parts: [32-block][quarter][column][16 bytes]
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int P = mx_parts(kElem<T>);
  const int nb = (a.k + 127) / 128 * 4, cols = (int)a.m * P;
  const int gb = kMxGemvWaves / kw, slot = wv / kw, kz = wv % kw;
  const int steps = nb / 4, ns = (steps + kw - 1) / kw, s0 = kz * ns;   // this wave's steps [s0, s0 + ns), as far as they exist
  const int g = lane >> 4, c16 = lane & 15;
  const int64_t groups = (a.n + 15) / 16;
  const uint8_t* wsc = a.w + (size_t)a.wrt * a.kt * 1024;
  const int kt = a.kt, ks = a.ks;

  // the ring of weights in flight: (group, step) pairs in the order of use
  u32x4 wr[kGemvAhead];
  int wsr[kGemvAhead];
  int64_t lbase = (int64_t)blockIdx.x * gb;
  int ls = 0;
  const uint8_t *wp, *sp;
  auto row_group = [&]() __attribute__((always_inline)) {
    // reads past the end repeat the last row group
    const int64_t q = min(lbase + slot, groups - 1), R = q >> 1;
    const int in = 32 * (g & 1) + 16 * (int)(q & 1) + c16;
    wp = a.w + (size_t)R * kt * 1024 + 16 * in;
    sp = wsc + (size_t)R * ks * 256 + 4 * in;
  };
  row_group();
  const int t0 = 2 * s0 + (g >> 1);
  auto issue = [&](int r) __attribute__((always_inline)) {
    // or the last k group: past the k groups x is zero (the last step's second
    // tile) or the step is not used
    const int t = min(t0 + 2 * ls, kt - 1);
    wr[r] = __builtin_nontemporal_load((const u32x4*)(wp + (size_t)t * 1024));
    wsr[r] = sp[(t >> 2) * 256 + (t & 3)];
    if (++ls == ns) {
      ls = 0;
      lbase += (int64_t)gridDim.x * gb;
      row_group();
    }
  };

  // The parts: four lanes to a 32-block, eight elements each. Loads return in
  // order, so x is asked for before the weights are.
  {
    const T* x = (const T*)a.x;
    const int items = (int)a.m * nb, unit = tid & 3;
    const bool vec = ((uintptr_t)x % (4 * sizeof(T))) == 0 && a.ldx % 4 == 0;
    for (int i0 = 0; i0 < items; i0 += kMxGemvWaves * 16) {
      const int it = i0 + (tid >> 2), ic = min(it, items - 1), r = ic / nb, kb = ic - r * nb;
      const int64_t c = (int64_t)kb * 32 + 8 * unit;
      float h[2][4];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (vec) load4<T, true>(x + r * a.ldx, c + 4 * q, a.k, h[q]);
        else load4<T, false>(x + r * a.ldx, c + 4 * q, a.k, h[q]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i0 == 0) {
#pragma unroll
        for (int q = 0; q < kGemvAhead; ++q) issue(q);
      }
      __builtin_amdgcn_sched_barrier(0);
      float u[8] = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
      inf_to_nan<T>(u);
      uint8_t* d = rec + ((size_t)(4 * kb + unit) * cols + r * P) * 16;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const u32x4 z = take_part(u);
        if (it < items) *(u32x4*)(d + 16 * p) = z;
      }
    }
  }
  __syncthreads();
  const int64_t iters = (groups + (int64_t)gridDim.x * gb - 1) / ((int64_t)gridDim.x * gb);
  const int64_t total = iters * ns;
  const uint8_t* xr[NC];   // this lane's part of the wave's first step
#pragma unroll
  for (int c = 0; c < NC; ++c) xr[c] = rec + ((size_t)(4 * s0 + g) * 4 * cols + min(16 * c + c16, cols - 1)) * 16;
  f32x4 acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  int64_t base = (int64_t)blockIdx.x * gb;
  int s = 0;
  for (int64_t i = 0; i < total; i += kGemvAhead) {
#pragma unroll
    for (int r = 0; r < kGemvAhead; ++r) {
      if (i + r >= total) break;
      if (s0 + s < steps) {
        const float scale = scale_of(wsr[r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bf16x8 w = expand8(wr[r][e], scale);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const u32x4 x = *(const u32x4*)(xr[c] + (size_t)(16 * s + e) * cols * 16);
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(bf16x8, x), acc[c], 0, 0, 0);
          }
        }
      }
      issue(r);
      if (++s < ns) continue;
      // the row groups' sums over the parts and over the waves that share them
      s = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          red[(wv * 16 + 4 * g + e) * RP + 16 * c + c16] = acc[c][e];
          acc[c][e] = 0.f;
        }
      __syncthreads();
      // kw lanes an output, each the parts of one wave
      const int outs = gb * 16 * (int)a.m, z = tid & (kw - 1);
      for (int o0 = 0; o0 < outs; o0 += 64 * kMxGemvWaves / kw) {
        const int o = o0 + tid / kw, oc = min(o, outs - 1);
        const int row = oc & 15, sl = (oc >> 4) & (gb - 1), mr = oc / (16 * gb);
        const float* q = red + ((sl * kw + z) * 16 + row) * RP + mr * P;
        float v = q[P - 1];
#pragma unroll
        for (int p = P - 2; p >= 0; --p) v += q[p];
        if (kw >= 2) v += dpp_mov<0xB1>(v);
        if (kw >= 4) v += dpp_mov<0x4E>(v);
        if (kw >= 8) v += dpp_mov<0x141>(v);
        const int64_t nrow = (base + sl) * 16 + row;
        if (z == 0 && o < outs && nrow < a.n) store_elem(a.y_elem, a.y, mr * a.ldy + nrow, v);
      }
      __syncthreads();
      base += (int64_t)gridDim.x * gb;
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: weights as the first operand (rows of the result), x as the
// second; a block computes BN features of BM rows over one slice of k, a wave
// NF x MF tiles of 32 x 32. Packed x goes with the weights as they are through the
// 32 x 32 x 64 MX instruction; parts of x through 32 x 32 x 16 bf16 ones, for which a
// wave expands its weights, eight a lane before each (a conversion makes two
// in 5 cycles, an instruction takes 32). The parts of a k group are further steps
// of the same sums.
// The operands lie in memory in operand order, so a stage (ST steps) goes to
// LDS as it is, by DMA, 1 KB an instruction, NS - 1 stages ahead of the one
// that is multiplied; one barrier a stage. In the largest tile of packed x
// four waves only copy, so that the others' matrix instructions do not queue
// behind a stage's 72 copies: 4096 x 8192 x 8192 140 -> 129 us (with one copying
// wave, which cannot start them fast enough, 136; with two 127). In 128 x 64
// blocks two do (300 x 8192 x 4096 15.6 -> 14.1 us, 187 x 13824 x 1152 8.2 -> 7.7). In the
// others, whose stages are short (128 x 32) or long in cycles (parts), the waves
// share the copies.
// With more than two stages every copying wave starts the same number (CPW) in
// every stage, so that the number in flight tells which stage has arrived.
// Bound by the matrix units and their power. Packed x: a loop on registers
// reaches 6.4 PFLOP/s on random operands (9.3 on constant ones: the clock
// falls to 1.6 GHz), 256 x 256 blocks 4.0 to 4.3 (4096 x 8192 x 8192, 128 to 136 us from box
// to box), of which 16 us are each block's start and the store of its results. 16 x 16 x 128
// instructions reach 4.6 in the loop. Blocks of half the size, two to a CU, and
// more stages measured no faster.
// Parts: 4000 x 8192 x 8192 bf16 401 to 466 us from box to box (1.15 to 1.34 PFLOP/s; a
// bf16 library product of 8192 x 8192 x 8192 reaches 1.19), 2048 x 13824 x 1152 f32, three
// parts, 170 to 180 us in 256 x 64 blocks (1.09 to 1.15 of them). 4000 x 8192 x 8192 with
// the making of the parts, one box: 256 x 256 blocks with waves of 64 features x 128 rows
// 417 us, of 128 x 64 423, four of 128 x 128 456, three stages 429; another: 430, two blocks of 256 x
// 128 a CU 435 to 452.
// ---------------------------------------------------------------------------
template <bool X4, int NF, int MF, int WN, int WM, int ST, int NS>
struct GemmShape {
  static constexpr int BN = 32 * NF * WN, BM = 32 * MF * WM, NW = WN * WM;
  static constexpr int XG = X4 ? 1024 : kMxPartBytes;          // bytes of a row group's x in a step
  static constexpr int WU = BN / 32 * ST;                      // DMA units of a stage's weights,
  static constexpr int XQ = BM / 32 * XG / 1024, XU = XQ * ST; // of a step's and a stage's x,
  static constexpr int GN = (BN + (X4 ? BM : 0)) / 32, SU = (GN + 3) / 4;   // and of the row groups' scale dwords
  static constexpr int COPIERS = !X4 ? 0 : NF * MF >= 8 ? 4 : NF * MF == 2 ? 2 : 0;   // waves that only copy
  static constexpr int THREADS = 64 * (NW + COPIERS), CW = COPIERS ? COPIERS : NW;
  static constexpr int CPW = (WU + CW - 1) / CW + (XU + CW - 1) / CW + (SU + CW - 1) / CW;
  static_assert(ST == 4 || ST == 2 || ST == 1, "a stage lies within four k groups, whose scale bytes are one dword");
  static_assert(X4 || ST < 4, "the steps of a stage are looked at one by one");
  // With two stages nothing is copied twice, and the scale dwords of four k
  // groups alternate between two places; else each stage brings its own.
  static constexpr bool ONCE = NS == 2;
  static constexpr int SS = ONCE ? 2 : NS;
  static_assert(NS == 2 || NS == 3, "stages");
  static_assert(BM / 32 <= kMxPadGroups + 1 || X4, "the parts are padded for the last block");
  static_assert(NS == 2 || CPW < 64, "what a wave can wait for");
};

// One DMA instruction: lane l's 16 bytes at src go to dst + 16 l. Inline asm,
// because the compiler would wait for every DMA in flight before any LDS read;
// the waits before the barrier that precedes the readers are written out.
__device__ __forceinline__ void dma16(const uint8_t* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                   __builtin_amdgcn_readfirstlane(dst)),
               "v"(src)
               : "memory", "m0");
}
// The same from a uniform address: lane l's 16 bytes are at base + off, off = 16 l.
__device__ __forceinline__ void dma16u(const uint8_t* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                   __builtin_amdgcn_readfirstlane(dst)),
               "v"(off), "s"(base)
               : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <bool X4, int NF, int MF, int WN, int WM, int ST, int NS, int OCC>
__global__ __launch_bounds__((GemmShape<X4, NF, MF, WN, WM, ST, NS>::THREADS), OCC) void k_mx4_gemm(Mx4LinearArgs a, int nbn, int nbm, int bm0) {
  typedef GemmShape<X4, NF, MF, WN, WM, ST, NS> S;
  __shared__ __align__(1024) uint8_t stage[NS][(S::WU + S::XU) * 1024];
  __shared__ __align__(1024) uint8_t sstage[S::SS][S::SU * 1024];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wv % WN, wm = wv / WN;
  // Tile order: the blocks with one value of blockIdx % 8 share an XCD and its
  // L2; they take a contiguous range of an order with the k slices slowest,
  // then groups of 4 tile rows, the rows fastest.
  constexpr int GROUP = 4;
  const int G = gridDim.x, xcd = blockIdx.x & 7;
  const int LL = xcd * (G >> 3) + min(xcd, G & 7) + (blockIdx.x >> 3);
  const int kz = LL / (nbn * nbm), L = LL - kz * (nbn * nbm);
  const int fm = L / (GROUP * nbn) * GROUP, gm = min(nbm - fm, GROUP), Lp = L % (GROUP * nbn);
  const int64_t bm = bm0 + fm + Lp % gm, bn = Lp / gm;
  const int t_lo = 4 * (int)((int64_t)a.ks * kz / a.kslices), t_hi = min(4 * (int)((int64_t)a.ks * (kz + 1) / a.kslices), a.kt);
  const uint8_t* x = (const uint8_t*)a.x;
  const uint8_t* wsc = a.w + (size_t)a.wrt * a.kt * 1024;
  const uint8_t* xsc = x + (size_t)a.xrt * a.kt * 1024;   // of packed x
  const int64_t rn0 = bn * (S::BN / 32), rm0 = bm * (S::BM / 32);   // first row groups
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&stage[0][0];
  const uint32_t slds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&sstage[0][0];
  // A step is a k group of packed x, a part of a k group of x otherwise: step
  // P t + p multiplies the weights of k group t by part p.
  const int P = X4 ? 1 : a.parts, u_lo = P * t_lo, u_hi = P * t_hi;
  // The lanes' sources at step 0. Row groups and k groups past the matrix
  // read its last ones, parts past the last row group what follows them; their
  // results are not stored, their x is not multiplied.
  constexpr int NWC = (S::WU + S::CW - 1) / S::CW, NXC = (S::XU + S::CW - 1) / S::CW, NSC = (S::SU + S::CW - 1) / S::CW;
  const int cw = S::COPIERS > 0 ? wv - S::NW : wv;
  const uint8_t *wsrc[NWC], *xsrc[NXC], *ssrc[NSC];
  const int kt = a.kt, ks = a.ks;
  const int64_t wlast = a.wrt - 1, xlast = a.xrt - 1;
  const size_t xstep = X4 ? 1024 : (size_t)a.xrt * S::XG;
#pragma unroll
  for (int i = 0; i < NWC; ++i) {
    const int u = min(i * S::CW + cw, S::WU - 1);
    wsrc[i] = a.w + (size_t)min(rn0 + u / ST, wlast) * kt * 1024 + 16 * lane;
  }
#pragma unroll
  for (int i = 0; i < NXC; ++i) {
    const int u = min(i * S::CW + cw, S::XU - 1);
    if constexpr (X4) xsrc[i] = x + (size_t)min(rm0 + u / ST, xlast) * kt * 1024 + 16 * lane;
    // the block's row groups of one step lie one after the other
    else xsrc[i] = x + (size_t)rm0 * S::XG + u % S::XQ * 1024 + 16 * lane;
  }
#pragma unroll
  for (int i = 0; i < NSC; ++i) {
    // 16 lanes a row group's 256 bytes of scales
    const int gi = min(4 * min(i * S::CW + cw, S::SU - 1) + (lane >> 4), S::GN - 1);
    ssrc[i] = (gi < S::BN / 32 ? wsc + (size_t)min(rn0 + gi, wlast) * ks * 256
                               : xsc + (size_t)min(rm0 + gi - S::BN / 32, xlast) * ks * 256) + 16 * (lane & 15);
  }
  // With two stages a wave waits for all its copies, and nothing is copied
  // twice. With more their number has to be the same in every stage: units are
  // fetched again where there are none left.
  int ct = t_lo, cp = 0;   // k group and part of the next step to copy
  auto copy = [&](int u0, int buf) __attribute__((always_inline)) {
    const uint32_t dst = lds + buf * ((S::WU + S::XU) * 1024);
    const int t = ct;
    const bool scales = !S::ONCE || ((t & 3) == 0 && cp == 0);
    int tq[ST];   // the steps' k groups
#pragma unroll
    for (int q = 0; q < ST; ++q) {
      tq[q] = ST == 1 ? ct : min(ct, kt - 1);
      if (X4 || ++cp == P) {
        cp = 0;
        ++ct;
      }
    }
#pragma unroll
    for (int i = 0; i < NWC; ++i) {
      const int u = min(i * S::CW + cw, S::WU - 1);
      int tw = tq[0];
#pragma unroll
      for (int q = 1; q < ST; ++q) tw = u % ST == q ? tq[q] : tw;
      if (!S::ONCE || S::WU % S::CW == 0 || i * S::CW + cw < S::WU) dma16(wsrc[i] + (size_t)tw * 1024, dst + 1024 * u);
    }
#pragma unroll
    for (int i = 0; i < NXC; ++i) {
      const int u = min(i * S::CW + cw, S::XU - 1), q = X4 ? u % ST : u / S::XQ;
      if (!S::ONCE || S::XU % S::CW == 0 || i * S::CW + cw < S::XU)
        dma16(xsrc[i] + (size_t)(ST == 1 ? u0 : min(u0 + q, kt * P - 1)) * xstep, dst + 1024 * (S::WU + u));
    }
    if (!scales) return;
#pragma unroll
    for (int i = 0; i < NSC; ++i) {
      const int u = min(i * S::CW + cw, S::SU - 1);
      if (!S::ONCE || i * S::CW + cw < S::SU) dma16(ssrc[i] + (t >> 2) * 256, slds + (S::ONCE ? (t >> 2) & 1 : buf) * (S::SU * 1024) + u * 1024);
    }
  };
  // Waits for the stage at step u: the copies of the stage behind it, if there
  // is one, may stay in flight.
  auto arrived = [&](int u) __attribute__((always_inline)) {
    if (NS == 2) wait_copies<0>();
    else if (u + ST < u_hi) wait_copies<S::CPW>();
    else wait_copies<0>();
  };
  int buf = 0, fill = NS - 1;
  if constexpr (S::COPIERS > 0) {
    if (wv >= S::NW) {
      // addresses in scalar registers (64-bit sums in every lane for each copy:
      // 147 us instead of 136 for the packed x above with one copying wave)
      constexpr int C = S::COPIERS, GW = S::BN / 32 / C, GX = S::BM / 32 / C, GS = S::SU / C;
      static_assert(X4 && GW * C * ST == S::WU && GX * C * ST == S::XU && GS * C == S::SU, "equal shares");
      const uint8_t *wb[GW], *xb[GX], *sb[GS];
#pragma unroll
      for (int i = 0; i < GW; ++i) wb[i] = a.w + (size_t)min(rn0 + cw * GW + i, wlast) * kt * 1024;
#pragma unroll
      for (int i = 0; i < GX; ++i) xb[i] = x + (size_t)min(rm0 + cw * GX + i, xlast) * kt * 1024;
#pragma unroll
      for (int i = 0; i < GS; ++i) {
        const int gi = 4 * (cw * GS + i) + (lane >> 4);
        sb[i] = (gi < S::BN / 32 ? wsc + (size_t)min(rn0 + gi, wlast) * ks * 256
                                 : xsc + (size_t)min(rm0 + gi - S::BN / 32, xlast) * ks * 256) + 16 * (lane & 15);
      }
      auto copy_share = [&](int t, int buf) __attribute__((always_inline)) {
        const uint32_t dst = lds + buf * ((S::WU + S::XU) * 1024);
#pragma unroll
        for (int q = 0; q < ST; ++q) {
          const int tq = ST == 1 ? t : min(t + q, kt - 1);
#pragma unroll
          for (int i = 0; i < GW; ++i)
            dma16u(wb[i] + (size_t)tq * 1024, 16 * lane, dst + 1024 * ((cw * GW + i) * ST + q));
#pragma unroll
          for (int i = 0; i < GX; ++i)
            dma16u(xb[i] + (size_t)tq * 1024, 16 * lane, dst + 1024 * (S::WU + (cw * GX + i) * ST + q));
        }
        if (S::ONCE && ST < 4 && (t & 3) != 0) return;
#pragma unroll
        for (int i = 0; i < GS; ++i)
          dma16(sb[i] + (t >> 2) * 256, slds + (S::ONCE ? (t >> 2) & 1 : buf) * (S::SU * 1024) + (cw * GS + i) * 1024);
      };
      __builtin_amdgcn_s_setprio(3);
#pragma unroll
      for (int i = 0; i < NS - 1; ++i)
        if (t_lo + i * ST < t_hi) copy_share(t_lo + i * ST, i);
      // the barriers of the waves that multiply, and the copies between them
      for (int t = t_lo; t < t_hi; t += ST) {
        arrived(t);
        __syncthreads();
        if (t + (NS - 1) * ST < t_hi) copy_share(t + (NS - 1) * ST, fill);
        fill = fill + 1 == NS ? 0 : fill + 1;
      }
      __syncthreads();
      return;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
      if (u_lo + i * ST < u_hi) copy(u_lo + i * ST, i);
  }
  f32x16 acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  int mt = t_lo, mp = 0;   // k group and part of the step to multiply
  for (int u = u_lo; u < u_hi; u += ST) {
    if (S::COPIERS == 0) arrived(u);
    __syncthreads();   // the stage has arrived for every wave, and every wave has read the one before
    if (S::COPIERS == 0 && u + (NS - 1) * ST < u_hi) copy(u + (NS - 1) * ST, fill);
    fill = fill + 1 == NS ? 0 : fill + 1;
    const uint8_t* ws = stage[buf] + 16 * lane;
    const uint8_t* xs = ws + S::WU * 1024;
    const uint32_t* sd = (const uint32_t*)sstage[S::ONCE ? (mt >> 2) & 1 : buf] + lane;
    buf = buf + 1 == NS ? 0 : buf + 1;
    int wd[NF], xd[MF];   // scale dwords: byte t % 4 is k group t's
#pragma unroll
    for (int i = 0; i < NF; ++i) wd[i] = sd[(wn * NF + i) * 64];
#pragma unroll
    for (int j = 0; j < MF; ++j) xd[j] = X4 ? sd[(S::BN / 32 + wm * MF + j) * 64] : 0;
#pragma unroll
    for (int q = 0; q < ST; ++q) {
      if (ST > 1 && u + q >= u_hi) break;
      u32x4 w[NF];
#pragma unroll
      for (int i = 0; i < NF; ++i) w[i] = *(const u32x4*)(ws + ((wn * NF + i) * ST + q) * 1024);
      const int sh = 8 * (mt & 3);
      if constexpr (X4) {
#pragma unroll
        for (int j = 0; j < MF; ++j) {
          const u32x4 v = *(const u32x4*)(xs + ((wm * MF + j) * ST + q) * 1024);
          const i32x8 b = {(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < NF; ++i) {
            const i32x8 wi = {(int)w[i][0], (int)w[i][1], (int)w[i][2], (int)w[i][3], 0, 0, 0, 0};
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wi, b, acc[i][j], kFp4, kFp4, 0, (uint32_t)wd[i] >> sh, 0,
                                                                        (uint32_t)xd[j] >> sh);
          }
        }
        ++mt;
      } else {
        float scale[NF];
#pragma unroll
        for (int i = 0; i < NF; ++i) scale[i] = scale_of(((uint32_t)wd[i] >> sh) & 255);
        // a quarter of each 32-block at a time: instruction e takes elements 8 e .. 8 e + 7 of both
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bf16x8 we[NF];
#pragma unroll
          for (int i = 0; i < NF; ++i) we[i] = expand8(w[i][e], scale[i]);
#pragma unroll
          for (int j = 0; j < MF; ++j) {
            const u32x4 v = *(const u32x4*)(xs + (q * S::XQ + (wm * MF + j) * 4 + e) * 1024);
#pragma unroll
            for (int i = 0; i < NF; ++i)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(we[i], __builtin_bit_cast(bf16x8, v), acc[i][j], 0, 0, 0);
          }
        }
        if (++mp == P) {
          mp = 0;
          ++mt;
        }
      }
    }
  }
  // A lane holds elements 4 e .. 4 e + 3 as features 8 e + 4 (lane / 32) .. of
  // row lane % 32: they change places in LDS, a wave HF tiles at a time, so that
  // whole lines of y are written. A slice of k leaves f32 sums.
  void* y = a.y;
  int64_t ldy = a.ldy;
  int elem = a.y_elem, vec = a.y_vec;
  if (a.kslices > 1) {
    y = a.partial + (size_t)kz * a.m * a.ldp;
    ldy = a.ldp;
    elem = ELEM_F32;
    vec = 1;
  }
  constexpr int ROOM = NS * (S::WU + S::XU) * 1024;
  constexpr int HF = NF > 1 && S::NW * 32 * 68 * 4 <= ROOM ? 2 : 1, PITCH = 32 * HF + 4;
  static_assert(S::NW * 32 * PITCH * 4 <= ROOM, "the stages hold a tile of each wave");
  float* tile = (float*)&stage[0][0] + wv * 32 * PITCH;
  __syncthreads();   // every wave has read its last stage
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    const int64_t row0 = (rm0 + wm * MF + j) * 32;
#pragma unroll
    for (int i0 = 0; i0 < NF; i0 += HF) {
      const int64_t f0 = (rn0 + wn * NF + i0) * 32;
#pragma unroll
      for (int i = 0; i < HF; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *(f32x4*)(tile + (lane & 31) * PITCH + 32 * i + 8 * e + 4 * (lane >> 5)) =
              f32x4{acc[i0 + i][j][4 * e], acc[i0 + i][j][4 * e + 1], acc[i0 + i][j][4 * e + 2], acc[i0 + i][j][4 * e + 3]};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      store_tile<32 * HF, PITCH>(elem, y, ldy, row0, f0, a.m, a.n, vec, tile, lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// The k slices' sums, added in order; four features a thread. Bound by their
// read (6.7 TB/s of many; 2.9 us of few).
__global__ __launch_bounds__(256) void k_mx4_join(Mx4LinearArgs a) {
  const int64_t f = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const int64_t row = blockIdx.y;
  if (f >= a.n) return;
  const float* p = a.partial + row * a.ldp + f;   // ldp is a multiple of 4: whole vectors
  f32x4 v = *(const f32x4*)p;
  for (int z = 1; z < a.kslices; ++z) v += *(const f32x4*)(p + (size_t)z * a.m * a.ldp);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (f + e < a.n) store_elem(a.y_elem, a.y, row * a.ldy + f + e, v[e]);
}

// Rows can be read n elements at once.
template <class T>
bool rows_aligned(const void* p, int64_t ld, int n) {
  return ((uintptr_t)p % (n * sizeof(T))) == 0 && ld % n == 0;
}

// A launch for each 2^23 row groups (a grid holds fewer than 2^32 threads):
// f(first row group, grid).
template <class F>
int by_row_groups(const Mx4Layout& L, F f) {
  constexpr int64_t MOST = 1 << 23;
  for (int64_t r0 = 0; r0 < L.rt; r0 += MOST) {
    f(r0, dim3((unsigned)std::min(L.rt - r0, MOST), (unsigned)L.ks));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

template <class T>
int quantize_t(const void* src, int64_t rows, int64_t k, int64_t ld, uint8_t* dst, hipStream_t s) {
  const Mx4Layout L = mx4_layout(rows, k);
  const bool vec = rows_aligned<T>(src, ld, 16 / (int)sizeof(T));
  return by_row_groups(L, [&](int64_t r0, dim3 grid) {
    if (vec) hipLaunchKernelGGL((k_mx4_quantize<T, true>), grid, dim3(256), 0, s, (const T*)src, rows, k, ld, dst, L, r0);
    else hipLaunchKernelGGL((k_mx4_quantize<T, false>), grid, dim3(256), 0, s, (const T*)src, rows, k, ld, dst, L, r0);
  });
}

template <class T>
int split_t(const void* src, int64_t rows, int64_t k, int64_t ld, uint8_t* dst, hipStream_t s) {
  const Mx4Layout L = mx4_layout(rows, k);
  const dim3 grid((unsigned)L.rt, (unsigned)L.kt);
  if (rows_aligned<T>(src, ld, 4))
    hipLaunchKernelGGL((k_mx_split<T, true>), grid, dim3(64), 0, s, (const T*)src, rows, k, ld, dst, L);
  else
    hipLaunchKernelGGL((k_mx_split<T, false>), grid, dim3(64), 0, s, (const T*)src, rows, k, ld, dst, L);
  return (int)hipGetLastError();
}

}  // namespace

int launch_mx4_quantize(int elem, const void* src, int64_t rows, int64_t k, int64_t ld, uint8_t* dst, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  switch (elem) {
    case ELEM_F32: return quantize_t<float>(src, rows, k, ld, dst, s);
    case ELEM_F16: return quantize_t<_Float16>(src, rows, k, ld, dst, s);
    case ELEM_BF16: return quantize_t<__bf16>(src, rows, k, ld, dst, s);
  }
  return (int)hipErrorInvalidValue;
}

int launch_mx4_dequant(const uint8_t* src, float* out, int64_t rows, int64_t k, int64_t ld, void* stream) {
  const Mx4Layout L = mx4_layout(rows, k);
  hipStream_t s = (hipStream_t)stream;
  const bool vec = rows_aligned<float>(out, ld, 4);
  return by_row_groups(L, [&](int64_t r0, dim3 grid) {
    if (vec) hipLaunchKernelGGL((k_mx4_dequant<true>), grid, dim3(256), 0, s, src, out, rows, k, ld, L, r0);
    else hipLaunchKernelGGL((k_mx4_dequant<false>), grid, dim3(256), 0, s, src, out, rows, k, ld, L, r0);
  });
}

int launch_mx_split(int elem, const void* src, int64_t rows, int64_t k, int64_t ld, uint8_t* dst, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  switch (elem) {
    case ELEM_F32: return split_t<float>(src, rows, k, ld, dst, s);
    case ELEM_F16: return split_t<_Float16>(src, rows, k, ld, dst, s);
    case ELEM_BF16: return split_t<__bf16>(src, rows, k, ld, dst, s);
  }
  return (int)hipErrorInvalidValue;
}

template <class T>
static int launch_gemv_t(const Mx4LinearArgs& a, hipStream_t s) {
  const int cols = (int)a.m * a.parts, kw = mx_gemv_waves(a.n, a.k);
  const int64_t groups = (a.n + 15) / 16;
  const size_t lds = mx_gemv_lds(cols, a.k);
  const int64_t blocks = (groups * kw + kMxGemvWaves - 1) / kMxGemvWaves;
  // every block makes all parts: one a CU, and two where each has several row
  // groups to go over and LDS holds both (more weights in flight)
  const int64_t most = blocks >= 1024 && lds <= 80 * 1024 ? 512 : 256;
  const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(64 * kMxGemvWaves);
  constexpr int MOST = (mx_parts(kElem<T>) * kMxGemvRows + 15) / 16;   // column tiles
  const int tiles = (cols + 15) / 16;
  if (tiles == 1) hipLaunchKernelGGL((k_mx4_gemv<T, 1>), grid, block, lds, s, a, kw);
  else if (tiles == 2) hipLaunchKernelGGL((k_mx4_gemv<T, 2>), grid, block, lds, s, a, kw);
  else if (tiles == 3 && MOST >= 3) hipLaunchKernelGGL((k_mx4_gemv<T, MOST >= 3 ? 3 : 2>), grid, block, lds, s, a, kw);
  else if (tiles == 4 && MOST >= 4) hipLaunchKernelGGL((k_mx4_gemv<T, MOST >= 4 ? 4 : 2>), grid, block, lds, s, a, kw);
  else return (int)hipErrorInvalidValue;
  return (int)hipGetLastError();
}

int launch_mx4_gemv(const Mx4LinearArgs& a, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  switch (a.x_elem) {
    case ELEM_F32: return launch_gemv_t<float>(a, s);
    case ELEM_F16: return launch_gemv_t<_Float16>(a, s);
    case ELEM_BF16: return launch_gemv_t<__bf16>(a, s);
  }
  return (int)hipErrorInvalidValue;
}

template <bool X4, int NF, int MF, int WN, int WM, int ST, int NS, int OCC>
static int launch_gemm_t(const Mx4LinearArgs& a, hipStream_t s) {
  typedef GemmShape<X4, NF, MF, WN, WM, ST, NS> S;
  const int64_t nbn = (a.n + S::BN - 1) / S::BN, nbm = (a.m + S::BM - 1) / S::BM;
  // a grid holds fewer than 2^32 threads: as many tile rows as fit in each
  // launch. 2^30 features are at most 2^23 tiles of 128, so that one row fits;
  // slices come only with few sums (kMx4MaxSums), in one launch.
  const int64_t rows = 0xffffffffll / S::THREADS / (nbn * a.kslices);
  if (rows < 1 || (a.kslices > 1 && rows < nbm)) return (int)hipErrorInvalidValue;
  hipError_t e = hipSuccess;
  for (int64_t b = 0; b < nbm && e == hipSuccess; b += rows) {
    const int64_t now = std::min(nbm - b, rows);
    hipLaunchKernelGGL((k_mx4_gemm<X4, NF, MF, WN, WM, ST, NS, OCC>), dim3((unsigned)(nbn * now * a.kslices)),
                       dim3(S::THREADS), 0, s, a, (int)nbn, (int)now, (int)b);
    e = hipGetLastError();
  }
  if (e != hipSuccess || a.kslices == 1) return (int)e;
  hipLaunchKernelGGL(k_mx4_join, dim3((unsigned)((a.n + 1023) / 1024), (unsigned)a.m), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

// The stages: 128 x 32 blocks, whose steps are short, copy two of them at a
// time, two stages ahead; packed x comes four k groups at a time.
int launch_mx4_gemm(const Mx4LinearArgs& a, bool packed, int tile, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (packed) {
    switch (tile) {
      case MT_256x256: return launch_gemm_t<true, 4, 2, 2, 4, 4, 2, 1>(a, s);
      case MT_128x64: return launch_gemm_t<true, 1, 2, 4, 1, 4, 2, 2>(a, s);
      case MT_128x32: return launch_gemm_t<true, 1, 1, 4, 1, 4, 3, 2>(a, s);
    }
  } else {
    switch (tile) {
      case MT_256x256: return launch_gemm_t<false, 2, 4, 4, 2, 1, 2, 1>(a, s);
      case MT_256x64: return launch_gemm_t<false, 2, 2, 4, 1, 1, 2, 2>(a, s);
      case MT_128x32: return launch_gemm_t<false, 1, 1, 4, 1, 2, 3, 2>(a, s);
    }
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
