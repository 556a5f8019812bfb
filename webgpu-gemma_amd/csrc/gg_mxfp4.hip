// gg_mxfp4.hip -- MXFP4 matrices on gfx950: quantisation, expansion, and
// products y = x W^T with W in MXFP4 and x in f32 / f16 / bf16 or MXFP4.
// The formats and layouts are described at Mx4Layout and mx_parts
// (gg_internal.h).
#include "gg_device.h"

namespace gg {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
constexpr int kFp6 = 2, kFp4 = 4;   // operand formats of the MX matrix instructions

template <class T>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) { return (float)((const T*)p)[i]; }

// Elements [c, c + 4) of a row of k elements, zeros past its end.
template <class T, bool VEC>
__device__ __forceinline__ void load4(const T* row, int64_t c, int64_t k, float (&v)[4]) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  if (VEC && c + 4 <= k) {
    const vec_t t = *(const vec_t*)(row + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i < k ? (float)row[c + i] : 0.f;
  }
}

__device__ __forceinline__ float group8_max(float x) {
  x = fmaxf(x, dpp_mov<0xB1>(x));
  x = fmaxf(x, dpp_mov<0x4E>(x));
  x = fmaxf(x, dpp_mov<0x141>(x));
  return x;
}

// ---------------------------------------------------------------------------
// Quantisation. A block takes 32 rows x 256 k (one group of scale dwords):
// a wave reads 256 consecutive elements of a row at a time, eight lanes to a
// 32-block; the codes go through LDS into operand order, so that both the
// reads and the 1 KB tiles written are whole lines.
// Scale byte: the exponent field of the block's largest magnitude less 2
// (floor(log2) - 2), at least 0; conversion to nearest, ties to even, values
// above 6 to 6. Bound by memory: reads the input once, writes 17/32 byte an
// element.
// ---------------------------------------------------------------------------
template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_mx4_quantize(const T* __restrict__ src, int64_t rows, int64_t k, int64_t ld,
                                                      uint8_t* __restrict__ dst, Mx4Layout L) {
  __shared__ __align__(16) uint16_t codes[256][8];   // [4 tiles x 64 lanes][16 bytes]
  __shared__ __align__(4) uint8_t scales[256];       // [64 lanes][4 tiles]
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = blockIdx.x;
  const int g = blockIdx.y;
  const int64_t c = (int64_t)g * 256 + 4 * lane;
  const int kb = lane >> 3, t = kb >> 1, b = kb & 1;   // 32-block, its tile and half
  float v[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = R * 32 + wv * 8 + i;
    if (r < rows) {
      load4<T, VEC>(src + r * ld, c, k, v[i]);
    } else {
      v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = wv * 8 + i;
    // the magnitudes' bits order as the magnitudes do, Inf and NaN on top
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) a = max(a, __float_as_uint(v[i][j]) & 0x7fffffffu);
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xf, 0xf, false));
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xf, 0xf, false));
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x141, 0xf, 0xf, false));
    const int ex = (int)(a >> 23);
    const int byte = ex == 255 ? 255 : max(ex - 2, 0);
    const float scale = __uint_as_float(byte ? (uint32_t)byte << 23 : 0x00400000u);   // byte 0: 2^-127
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][0], v[i][1], scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][2], v[i][3], scale, 1);
    if (byte == 255) q = 0;   // Inf or NaN in the block: its scale says NaN
    const int l = 32 * b + row;
    codes[t * 64 + l][lane & 7] = (uint16_t)q;
    if ((lane & 7) == 0) scales[4 * l + t] = (uint8_t)byte;
  }
  __syncthreads();
  if (g * 4 + wv < L.kt)
    *(u32x4*)(dst + ((size_t)R * L.kt + g * 4 + wv) * 1024 + 16 * lane) = *(const u32x4*)codes[wv * 64 + lane];
  if (wv == 0)
    *(uint32_t*)(dst + L.codes() + ((size_t)R * L.ks + g) * 256 + 4 * lane) = *(const uint32_t*)(scales + 4 * lane);
}

// ---------------------------------------------------------------------------
// Expansion to f32, the same tile the other way: each value is its 4-bit
// element times 2^(byte - 127), NaN where the byte is 255.
// ---------------------------------------------------------------------------
template <bool VEC>
__global__ __launch_bounds__(256) void k_mx4_dequant(const uint8_t* __restrict__ src, float* __restrict__ out,
                                                     int64_t rows, int64_t k, int64_t ld, Mx4Layout L) {
  __shared__ __align__(16) uint16_t codes[256][8];
  __shared__ __align__(4) uint8_t scales[256];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = blockIdx.x;
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
    if (r >= rows || c >= k) continue;
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
    float* d = out + r * ld + c;
    if (VEC && c + 4 <= k) {
      *(f32x4*)d = o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < k) d[j] = o[j];
    }
  }
}

// ---------------------------------------------------------------------------
// Activations in parts (mx_parts). A block of 32 with largest magnitude in
// [2^e, 2^(e+1)): scale byte e + 127, at least 21 so that every part's is at
// least 1, 255 when the block holds an Inf or a NaN (its row's results are
// NaN). part_round: u to the nearest multiple of 1/8 for |u| <= 2.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float part_round(float u) { return (u + 1572864.0f) - 1572864.0f; }   // 1.5 2^20: ulp 1/8
__device__ __forceinline__ int parts_byte(uint32_t amax_bits) {
  const int ex = (int)(amax_bits >> 23);
  return max(ex, 1 + 5 * (kMxMaxParts - 1));
}

// 32 rows x 256 k of a row-major matrix -> parts; thread tid owns the 32-block
// of lane tid % 64 of tile tid / 64.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_mx_split(const T* __restrict__ src, int64_t rows, int64_t k, int64_t ld,
                                                  int parts, uint8_t* __restrict__ dst, Mx4Layout L) {
  constexpr int kPitch = 257;   // a thread reads its row's block: 32 rows x 2 blocks fall on 64 banks
  __shared__ float xs[32 * kPitch];
  __shared__ __align__(4) uint8_t scales[256];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = blockIdx.x;
  const int g = blockIdx.y;
  const int64_t c = (int64_t)g * 256 + 4 * lane;
  float v[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = R * 32 + wv * 8 + i;
    if (r < rows) {
      load4<T, VEC>(src + r * ld, c, k, v[i]);
    } else {
      v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) xs[(wv * 8 + i) * kPitch + 4 * lane + j] = v[i][j];
  __syncthreads();
  const float* x = xs + (lane & 31) * kPitch + 64 * wv + 32 * (lane >> 5);
  f32x16 ev, od;   // even and odd elements: the conversion interleaves its operands
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    ev[i] = x[2 * i];
    od[i] = x[2 * i + 1];
    a = max(a, max(__float_as_uint(ev[i]) & 0x7fffffffu, __float_as_uint(od[i]) & 0x7fffffffu));
  }
  const int byte = parts_byte(a);
  scales[4 * lane + wv] = (uint8_t)byte;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    ev[i] = ldexpf(ev[i], 127 - byte);
    od[i] = ldexpf(od[i], 127 - byte);
  }
  const int t = g * 4 + wv;
  uint8_t* out = dst + ((size_t)R * L.kt + t) * parts * kMxPartBytes;
  for (int p = 0; p < parts; ++p) {
    f32x16 qe, qo;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      qe[i] = part_round(ev[i]);
      qo[i] = part_round(od[i]);
      ev[i] = (ev[i] - qe[i]) * 32.0f;
      od[i] = (od[i] - qo[i]) * 32.0f;
    }
    const u32x6 z = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(qe, qo, 1.0f);
    if (t < L.kt) {
      *(u32x4*)(out + p * kMxPartBytes + 16 * lane) = u32x4{z[0], z[1], z[2], z[3]};
      *(u32x2*)(out + p * kMxPartBytes + 1024 + 8 * lane) = u32x2{z[4], z[5]};
    }
  }
  __syncthreads();
  if (wv == 0)
    *(uint32_t*)(dst + (size_t)L.rt * L.kt * parts * kMxPartBytes + ((size_t)R * L.ks + g) * 256 + 4 * lane) =
        *(const uint32_t*)(scales + 4 * lane);
}

template <class T>
__device__ __forceinline__ void store_y(void* y, int64_t i, float v) { ((T*)y)[i] = (T)v; }
__device__ __forceinline__ void store_elem(int elem, void* y, int64_t i, float v) {
  if (elem == ELEM_F32) store_y<float>(y, i, v);
  else if (elem == ELEM_F16) store_y<_Float16>(y, i, v);
  else store_y<__bf16>(y, i, v);
}

// ---------------------------------------------------------------------------
// Few rows: m x parts <= 16 columns of the 16 x 16 x 128 matrix instruction,
// column r parts + p holding part p of row r, so that one instruction
// multiplies 16 weight rows x 128 k by every part at once and the sum over
// the parts is taken once, at the end, in f32. The parts are made in LDS by
// every block (k x m values), the weights go from memory to registers.
// A wave takes 16 weight rows; `kw` waves share their k.
// Bound by the read of the weights (17/32 byte each).
// ---------------------------------------------------------------------------
template <class T>
__device__ void gemv_parts(const Mx4LinearArgs& a, int nb, int cols, uint8_t* xs, uint8_t* sc) {
  // eight lanes to a 32-block, four elements each
  const T* x = (const T*)a.x;
  const int tid = threadIdx.x, P = a.parts, unit = tid & 7;
  const int items = (int)a.m * nb;
  for (int it = tid >> 3; it < items; it += blockDim.x >> 3) {
    const int r = it / nb, kb = it - r * nb;
    const int64_t c = (int64_t)kb * 32 + 4 * unit;
    float v[4];
    load4<T, false>(x + r * a.ldx, c, a.k, v);
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = max(mx, __float_as_uint(v[j]) & 0x7fffffffu);
    mx = max(mx, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mx, 0xB1, 0xf, 0xf, false));
    mx = max(mx, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mx, 0x4E, 0xf, 0xf, false));
    mx = max(mx, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mx, 0x141, 0xf, 0xf, false));
    const int byte = parts_byte(mx);
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = ldexpf(v[j], 127 - byte);
    for (int p = 0; p < P; ++p) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float q = part_round(u[j]);
        // e2m3 code of d / 8, d = 0..16, is d itself; bit 5 is the sign
        const uint32_t code = (uint32_t)fabsf(q * 8.0f) | (q < 0.f ? 32u : 0u);
        w |= (code & 63u) << (6 * j);
        u[j] = (u[j] - q) * 32.0f;
      }
      uint8_t* d = xs + ((size_t)kb * cols + r * P + p) * 24 + 3 * unit;
      d[0] = (uint8_t)w;
      d[1] = (uint8_t)(w >> 8);
      d[2] = (uint8_t)(w >> 16);
      if (unit == 0) sc[kb * cols + r * P + p] = (uint8_t)(byte == 255 ? 255 : byte - 5 * p);
    }
  }
}

constexpr int kGemvWaves = 8;
__global__ __launch_bounds__(64 * kGemvWaves) void k_mx4_gemv(Mx4LinearArgs a, int kw) {
  extern __shared__ uint8_t lds[];
  __shared__ float red[kGemvWaves][16][17];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = (a.k + 127) / 128 * 4, cols = (int)a.m * a.parts;
  uint8_t* xs = lds;
  uint8_t* sc = lds + (size_t)nb * cols * 24;
  if (a.x_elem == ELEM_F32) gemv_parts<float>(a, nb, cols, xs, sc);
  else if (a.x_elem == ELEM_F16) gemv_parts<_Float16>(a, nb, cols, xs, sc);
  else gemv_parts<__bf16>(a, nb, cols, xs, sc);
  __syncthreads();
  const int gb = kGemvWaves / kw, slot = wv / kw, kz = wv % kw;
  const int steps = nb / 4, s0 = steps * kz / kw, s1 = steps * (kz + 1) / kw;
  const int g = lane >> 4, c16 = lane & 15, col = min(c16, cols - 1);
  const int64_t groups = (a.n + 15) / 16;
  const uint8_t* wsc = a.w + (size_t)a.wrt * a.kt * 1024;
  for (int64_t base = (int64_t)blockIdx.x * gb; base < groups; base += (int64_t)gridDim.x * gb) {
    const int64_t q = min(base + slot, groups - 1), R = q >> 1;
    const int in = 32 * (g & 1) + 16 * (int)(q & 1) + c16;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; ++s) {
      // the last step's second tile may lie past the matrix: its x is zero,
      // the tile read instead is the last one
      const int t = min(2 * s + (g >> 1), a.kt - 1);
      const u32x4 w4 = *(const u32x4*)(a.w + ((size_t)R * a.kt + t) * 1024 + 16 * in);
      const int ws = wsc[((size_t)R * a.ks + (t >> 2)) * 256 + 4 * in + (t & 3)];
      const uint8_t* xp = xs + ((size_t)(4 * s + g) * cols + col) * 24;
      const u32x2 x0 = *(const u32x2*)xp, x1 = *(const u32x2*)(xp + 8), x2 = *(const u32x2*)(xp + 16);
      const int xsv = sc[(4 * s + g) * cols + col];
      const i32x8 wa = {(int)w4[0], (int)w4[1], (int)w4[2], (int)w4[3], 0, 0, 0, 0};
      const i32x8 xb = {(int)x0[0], (int)x0[1], (int)x1[0], (int)x1[1], (int)x2[0], (int)x2[1], 0, 0};
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc, kFp4, kFp6, 0, ws, 0, xsv);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wv][4 * g + r][c16] = acc[r];
    __syncthreads();
    for (int i = tid; i < gb * 16 * (int)a.m; i += 64 * kGemvWaves) {
      const int row = i % 16, sl = (i / 16) % gb, mr = i / (16 * gb);
      const int64_t nrow = (base + sl) * 16 + row;
      if (nrow >= a.n) continue;
      float v = 0.f;
      for (int p = a.parts - 1; p >= 0; --p)
        for (int z = 0; z < kw; ++z) v += red[sl * kw + z][row][mr * a.parts + p];
      store_elem(a.y_elem, a.y, mr * a.ldy + nrow, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: 32 x 32 x 64 matrix instructions, weights as the first operand
// (rows of the result), x as the second. A wave computes NF x MF tiles; the
// operands come from memory in operand order.
// ---------------------------------------------------------------------------
template <bool X4, int NF, int MF, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM) void k_mx4_gemm(Mx4LinearArgs a, int nbn, int nbm) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wv % WN, wm = wv / WN;
  const int64_t bn = blockIdx.x % nbn, bm = blockIdx.x / nbn;
  const int P = a.parts;
  int64_t rn[NF], rm[MF];
#pragma unroll
  for (int i = 0; i < NF; ++i) rn[i] = min((bn * WN + wn) * NF + i, a.wrt - 1);
#pragma unroll
  for (int j = 0; j < MF; ++j) rm[j] = min((bm * WM + wm) * MF + j, a.xrt - 1);
  const uint8_t* x = (const uint8_t*)a.x;
  const uint8_t* wsc = a.w + (size_t)a.wrt * a.kt * 1024;
  const uint8_t* xsc = x + (size_t)a.xrt * a.kt * (X4 ? 1024 : P * kMxPartBytes);
  f32x16 acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  for (int t = 0; t < a.kt; ++t) {
    i32x8 w[NF];
    int ws[NF], xs[MF];
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const u32x4 q = *(const u32x4*)(a.w + ((size_t)rn[i] * a.kt + t) * 1024 + 16 * lane);
      w[i] = i32x8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
      ws[i] = wsc[((size_t)rn[i] * a.ks + (t >> 2)) * 256 + 4 * lane + (t & 3)];
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) xs[j] = xsc[((size_t)rm[j] * a.ks + (t >> 2)) * 256 + 4 * lane + (t & 3)];
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int j = 0; j < MF; ++j) {
        i32x8 b;
        if constexpr (X4) {
          const u32x4 q = *(const u32x4*)(x + ((size_t)rm[j] * a.kt + t) * 1024 + 16 * lane);
          b = i32x8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
        } else {
          const uint8_t* xp = x + (((size_t)rm[j] * a.kt + t) * P + p) * kMxPartBytes;
          const u32x4 q = *(const u32x4*)(xp + 16 * lane);
          const u32x2 h = *(const u32x2*)(xp + 1024 + 8 * lane);
          b = i32x8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], (int)h[0], (int)h[1], 0, 0};
        }
        const int s = xs[j] == 255 ? 255 : xs[j] - 5 * p;
#pragma unroll
        for (int i = 0; i < NF; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i], b, acc[i][j], kFp4, X4 ? kFp4 : kFp6, 0,
                                                                      ws[i], 0, s);
      }
    }
  }
  // lane: result column lane % 32 (a row of y); elements 4 e .. 4 e + 3 are
  // features 8 e + 4 (lane / 32) ..
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    const int64_t row = (((bm * WM + wm) * MF) + j) * 32 + (lane & 31);
    if (row >= a.m) continue;
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t f = (((bn * WN + wn) * NF) + i) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (f < a.n) store_elem(a.y_elem, a.y, row * a.ldy + f, acc[i][j][e]);
      }
  }
}

template <class T>
bool aligned4(const void* p, int64_t ld) {
  return ((uintptr_t)p % (4 * sizeof(T))) == 0 && (ld * sizeof(T)) % (4 * sizeof(T)) == 0;
}

template <class T>
int quantize_t(const void* src, int64_t rows, int64_t k, int64_t ld, uint8_t* dst, hipStream_t s) {
  const Mx4Layout L = mx4_layout(rows, k);
  const dim3 grid((unsigned)L.rt, (unsigned)L.ks);
  if (aligned4<T>(src, ld))
    hipLaunchKernelGGL((k_mx4_quantize<T, true>), grid, dim3(256), 0, s, (const T*)src, rows, k, ld, dst, L);
  else
    hipLaunchKernelGGL((k_mx4_quantize<T, false>), grid, dim3(256), 0, s, (const T*)src, rows, k, ld, dst, L);
  return (int)hipGetLastError();
}

template <class T>
int split_t(const void* src, int64_t rows, int64_t k, int64_t ld, int parts, uint8_t* dst, hipStream_t s) {
  const Mx4Layout L = mx4_layout(rows, k);
  const dim3 grid((unsigned)L.rt, (unsigned)L.ks);
  if (aligned4<T>(src, ld))
    hipLaunchKernelGGL((k_mx_split<T, true>), grid, dim3(256), 0, s, (const T*)src, rows, k, ld, parts, dst, L);
  else
    hipLaunchKernelGGL((k_mx_split<T, false>), grid, dim3(256), 0, s, (const T*)src, rows, k, ld, parts, dst, L);
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
  const dim3 grid((unsigned)L.rt, (unsigned)L.ks);
  hipStream_t s = (hipStream_t)stream;
  if (aligned4<float>(out, ld))
    hipLaunchKernelGGL((k_mx4_dequant<true>), grid, dim3(256), 0, s, src, out, rows, k, ld, L);
  else
    hipLaunchKernelGGL((k_mx4_dequant<false>), grid, dim3(256), 0, s, src, out, rows, k, ld, L);
  return (int)hipGetLastError();
}

int launch_mx_split(int elem, const void* src, int64_t rows, int64_t k, int64_t ld, int parts, uint8_t* dst,
                    void* stream) {
  hipStream_t s = (hipStream_t)stream;
  switch (elem) {
    case ELEM_F32: return split_t<float>(src, rows, k, ld, parts, dst, s);
    case ELEM_F16: return split_t<_Float16>(src, rows, k, ld, parts, dst, s);
    case ELEM_BF16: return split_t<__bf16>(src, rows, k, ld, parts, dst, s);
  }
  return (int)hipErrorInvalidValue;
}

int launch_mx4_gemv(const Mx4LinearArgs& a, void* stream) {
  const int cols = (int)a.m * a.parts;
  const size_t lds = mx_gemv_lds(cols, a.k);
  const int64_t groups = (a.n + 15) / 16;
  int kw = 8;   // waves that share 16 rows' k: as many as leave 512 blocks busy
  while (kw > 1 && groups * kw > 8 * 512) kw >>= 1;
  const int64_t blocks = (groups * kw + kGemvWaves - 1) / kGemvWaves;
  hipLaunchKernelGGL(k_mx4_gemv, dim3((unsigned)(blocks < 512 ? blocks : 512)), dim3(64 * kGemvWaves), lds,
                     (hipStream_t)stream, a, kw);
  return (int)hipGetLastError();
}

int launch_mx4_gemm(const Mx4LinearArgs& a, bool x_mx4, void* stream) {
  constexpr int NF = 2, MF = 2, WN = 2, WM = 2;
  const int64_t nbn = (a.wrt + NF * WN - 1) / (NF * WN), nbm = (a.xrt + MF * WM - 1) / (MF * WM);
  if (nbn * nbm > 0x7fffffffll) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)(nbn * nbm)), block(64 * WN * WM);
  if (x_mx4)
    hipLaunchKernelGGL((k_mx4_gemm<true, NF, MF, WN, WM>), grid, block, 0, (hipStream_t)stream, a, (int)nbn, (int)nbm);
  else
    hipLaunchKernelGGL((k_mx4_gemm<false, NF, MF, WN, WM>), grid, block, 0, (hipStream_t)stream, a, (int)nbn, (int)nbm);
  return (int)hipGetLastError();
}

}  // namespace gg
