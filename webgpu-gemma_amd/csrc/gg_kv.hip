// gg_kv.hip -- new rows of a QKV product into K/V pages (RMS norm of the heads,
// rotation, 16 or 8 bits), and the values of pages back into rows.
//
//   y = x w / sqrt(mean x^2 + eps);  a = p theta^(-2j/D):
//   (y_j, y_{j+D/2}) -> (y_j cos a - y_{j+D/2} sin a, y_{j+D/2} cos a + y_j sin a)
//
// All of it is f64: a stored value is the formula's, rounded once. In f32 a value
// next to a border of the 8-bit format lands on its other side now and then, a
// whole step of 2^-4 away, and the angle of position 10^6 is off by 2^-5.
// 4380 rows of 48 heads of 128, bf16 to bf16 queries and 8-bit pages: 38 us, 98 MB at 2.6
// TB/s, a block being a row's chain of sequence, angles (one wave's) and heads in
// turn; v past the f64 and a shorter rounding took 40. Back into rows 9 us.
#include "gg_kv_device.h"

namespace gg {

namespace {

// f64 -> f32 towards zero with the last bit set where anything is cut off:
// rounding that to fewer bits gives what rounding the f64 value would.
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  uint32_t b = __float_as_uint(f);
  const double back = (double)f;
  if (back != x && fabs(x) < 0x1p128) {   // no NaN either
    if (fabs(back) > fabs(x)) b -= 1;     // from infinity too: to the largest f32, which is odd
    b |= 1;
  }
  return __uint_as_float(b);
}

template <class T>
__device__ __forceinline__ void load4(const T* p, bool vec, double (&x)[4]) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  if (vec) {
    const vec_t t = *(const vec_t*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (double)(float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (double)(float)p[i];
  }
}
template <class T>
__device__ __forceinline__ void store4(T* p, bool vec, const double (&x)[4]) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  vec_t t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) t[i] = (float)x[i];
    else t[i] = (T)to_odd(x[i]);
  }
  if (vec) {
    *(vec_t*)p = t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = t[i];
  }
}

__device__ __forceinline__ uint32_t fp8x4(const float (&f)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
}

// One block per row (and part of its heads). A head is held by D / 8 lanes of a
// group of G: values 4 j .. 4 j + 3 of each half, so that a rotation needs no
// other lane.
template <int KV, class T, class TQ, int G>
__global__ __launch_bounds__(256) void k_kv_store(KvStoreArgs a) {
  __shared__ double turn[kKvMaxDim / 2][2];
  const int tid = threadIdx.x, row = a.row0 + blockIdx.x;
  const int D = a.kv.dim, half = D / 2;
  const int heads = a.n_q + 2 * a.kv.n_kv;
  const int group = blockIdx.y * (256 / G) + tid / G, j = 4 * (tid % G), step = gridDim.y * (256 / G);
  const bool on = j < half;
  // the first head's values are on their way while the position is looked up
  auto source = [&](int h) __attribute__((always_inline)) {
    if (h < a.n_q) return (const T*)a.q + row * a.ldq + h * D;
    if (h < a.n_q + a.kv.n_kv) return (const T*)a.k + row * a.ldk + (h - a.n_q) * D;
    return (const T*)a.v + row * a.ldv + (h - a.n_q - a.kv.n_kv) * D;
  };
  double lo[4] = {}, hi[4] = {};
  if (group < heads && on) {
    load4(source(group) + j, a.vec, lo);
    load4(source(group) + half + j, a.vec, hi);
  }
  KvSeq sq;
  const int s = kv_seq_of(a.kv, row, &sq);
  if (s < 0) return;   // the same in all of the block
  const int pos = sq.len - sq.rows + (row - sq.first);
  KvPlace at{};
  const bool placed = pos >= 0 && pos < a.kv.places && kv_place(a.kv, s, pos, &at);
  if (a.rotate) {
    if (tid < half) {
      // the angle in turns, 1 / (2 pi) = 2^-2.651496129472319
      double t = pos * exp2(-(2.0 * tid / D) * a.log2_theta - 2.6514961294723187981);
      t -= rint(t);
      sincospi(2.0 * t, &turn[tid][1], &turn[tid][0]);
    }
    __syncthreads();
  }
  for (int h = group; h < heads; h += step) {
    if (h != group && on) {
      load4(source(h) + j, a.vec, lo);
      load4(source(h) + half + j, a.vec, hi);
    }
    const bool is_v = h >= a.n_q + a.kv.n_kv, is_q = h < a.n_q;
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (!is_v && w) {   // the same in all of a head's lanes
      double ss = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fma(lo[i], lo[i], fma(hi[i], hi[i], ss));
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, G);
      const double r = 1.0 / sqrt(ss / D + a.eps);
      if (on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] *= r * w[j + i];
          hi[i] *= r * w[half + j + i];
        }
      }
    }
    if (!is_v && a.rotate && on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double c = turn[j + i][0], n = turn[j + i][1], x = lo[i], y = hi[i];
        lo[i] = x * c - y * n;
        hi[i] = y * c + x * n;
      }
    }
    if (is_q) {
      if (on) {
        TQ* o = (TQ*)a.q_out + row * a.ldqo + (long long)h * D + j;
        const bool v = a.vec_q;
        store4(o, v, lo);
        store4(o + half, v, hi);
      }
      continue;
    }
    const int head = h - a.n_q - (is_v ? a.kv.n_kv : 0);
    void* base = is_v ? a.kv.v : a.kv.k;
    if constexpr (KV != KV_E4M3) {
      typedef typename std::conditional<KV == KV_BF16, __bf16, _Float16>::type C;
      if (on && placed) {
        C* o = (C*)base + kv_offset(a.kv, at, head) + j;
        store4(o, true, lo);
        store4(o + half, true, hi);
      }
    } else {
      float f[2][4];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[0][i] = to_odd(lo[i]);
        f[1][i] = to_odd(hi[i]);
        if (on) top = max(max(top, __float_as_uint(f[0][i]) & 0x7fffffffu), __float_as_uint(f[1][i]) & 0x7fffffffu);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, G));
      // the least e with top <= 448 2^e = 1.75 2^(e + 8); a value cut to odd stays above
      const int e = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
      const bool bad = top >= 0x7f800000u;
      const float inv = __uint_as_float((uint32_t)(127 - e) << 23);   // e is at most 120
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[0][i] = bad ? 0.f : f[0][i] * inv;
        f[1][i] = bad ? 0.f : f[1][i] * inv;
      }
      if (placed) {
        if (on) {
          uint8_t* o = (uint8_t*)base + kv_offset(a.kv, at, head) + j;
          *(uint32_t*)o = fp8x4(f[0]);
          *(uint32_t*)(o + half) = fp8x4(f[1]);
        }
        if (j == 0)
          (is_v ? a.kv.v_scale : a.kv.k_scale)[kv_scale_at(a.kv, at, head)] = bad ? NAN : __uint_as_float((uint32_t)(127 + e) << 23);
      }
    }
  }
}

// One block per row: eight values a thread.
template <int KV, class T>
__global__ __launch_bounds__(256) void k_kv_load(KvLoadArgs a) {
  const int row = a.row0 + blockIdx.x, D = a.kv.dim, per = D / 8, units = 2 * a.kv.n_kv * per;
  KvSeq sq;
  const int s = kv_seq_of(a.kv, row, &sq);
  if (s < 0) return;
  const int pos = sq.len - sq.rows + (row - sq.first);
  KvPlace at{};
  const bool placed = pos >= 0 && pos < a.kv.places && kv_place(a.kv, s, pos, &at);
  for (int u = threadIdx.x; u < units; u += 256) {
    const int h = u / per, e = 8 * (u % per);
    const bool is_v = h >= a.kv.n_kv;
    const int head = is_v ? h - a.kv.n_kv : h;
    T* out = (T*)(is_v ? a.v : a.k);
    if (!out) continue;
    out += row * (is_v ? a.ldv : a.ldk) + head * D + e;
    float f[8] = {};
    if (placed) {
      const long long o = kv_offset(a.kv, at, head) + e;
      const void* base = is_v ? a.kv.v : a.kv.k;
      if constexpr (KV == KV_E4M3) {
        const float sc = (is_v ? a.kv.v_scale : a.kv.k_scale)[kv_scale_at(a.kv, at, head)];
        const uint2 w = *(const uint2*)((const uint8_t*)base + o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = i < 4 ? w.x : w.y;
          f[i] = sc * (i % 4 == 0 ? __builtin_amdgcn_cvt_f32_fp8(x, 0) : i % 4 == 1 ? __builtin_amdgcn_cvt_f32_fp8(x, 1)
                       : i % 4 == 2 ? __builtin_amdgcn_cvt_f32_fp8(x, 2) : __builtin_amdgcn_cvt_f32_fp8(x, 3));
        }
      } else {
        typedef typename std::conditional<KV == KV_BF16, __bf16, _Float16>::type C;
        typedef C vec_t __attribute__((ext_vector_type(8)));
        const vec_t t = *(const vec_t*)((const C*)base + o);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)t[i];
      }
    }
    if (((uintptr_t)out & 15) == 0) {
      constexpr int V = 16 / sizeof(T);
      typedef T vec_t __attribute__((ext_vector_type(V)));
#pragma unroll
      for (int i = 0; i < 8; i += V) {
        vec_t t;
#pragma unroll
        for (int k = 0; k < V; ++k) t[k] = (T)f[i + k];
        *(vec_t*)(out + i) = t;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = (T)f[i];
    }
  }
}

constexpr int kMostRows = 1 << 22;   // of a launch: a grid holds fewer than 2^32 threads

template <int KV, class T, class TQ>
int store_g(KvStoreArgs a, hipStream_t s) {
  const int lanes = a.kv.dim / 8, heads = a.n_q + 2 * a.kv.n_kv;
  for (int r = 0; r < a.kv.n_rows; r += kMostRows) {
    a.row0 = r;
    const int rows = a.kv.n_rows - r < kMostRows ? a.kv.n_rows - r : kMostRows;
    const auto go = [&](auto kernel, int G) {
      const int each = 256 / G, parts = rows < 512 ? (heads + each - 1) / each : 1;
      hipLaunchKernelGGL(kernel, dim3(rows, parts), dim3(256), 0, s, a);
    };
    if (lanes <= 8) go(k_kv_store<KV, T, TQ, 8>, 8);
    else if (lanes <= 16) go(k_kv_store<KV, T, TQ, 16>, 16);
    else go(k_kv_store<KV, T, TQ, 32>, 32);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}
template <int KV, class T>
int store_q(int q_elem, const KvStoreArgs& a, hipStream_t s) {
  switch (q_elem) {
    case ELEM_F32: return store_g<KV, T, float>(a, s);
    case ELEM_F16: return store_g<KV, T, _Float16>(a, s);
    case ELEM_BF16: return store_g<KV, T, __bf16>(a, s);
  }
  return (int)hipErrorInvalidValue;
}
template <int KV>
int store_t(int elem, int q_elem, const KvStoreArgs& a, hipStream_t s) {
  switch (elem) {
    case ELEM_F32: return store_q<KV, float>(q_elem, a, s);
    case ELEM_F16: return store_q<KV, _Float16>(q_elem, a, s);
    case ELEM_BF16: return store_q<KV, __bf16>(q_elem, a, s);
  }
  return (int)hipErrorInvalidValue;
}

template <int KV, class T>
int load_r(KvLoadArgs a, hipStream_t s) {
  for (int r = 0; r < a.kv.n_rows; r += kMostRows) {
    a.row0 = r;
    const int rows = a.kv.n_rows - r < kMostRows ? a.kv.n_rows - r : kMostRows;
    hipLaunchKernelGGL((k_kv_load<KV, T>), dim3(rows), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}
template <int KV>
int load_t(int elem, const KvLoadArgs& a, hipStream_t s) {
  switch (elem) {
    case ELEM_F32: return load_r<KV, float>(a, s);
    case ELEM_F16: return load_r<KV, _Float16>(a, s);
    case ELEM_BF16: return load_r<KV, __bf16>(a, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace

int launch_kv_store(int kv_type, int elem, int q_elem, const KvStoreArgs& a, void* stream) {
  switch (kv_type) {
    case KV_BF16: return store_t<KV_BF16>(elem, q_elem, a, (hipStream_t)stream);
    case KV_F16: return store_t<KV_F16>(elem, q_elem, a, (hipStream_t)stream);
    case KV_E4M3: return store_t<KV_E4M3>(elem, q_elem, a, (hipStream_t)stream);
  }
  return (int)hipErrorInvalidValue;
}
int launch_kv_load(int kv_type, int elem, const KvLoadArgs& a, void* stream) {
  switch (kv_type) {
    case KV_BF16: return load_t<KV_BF16>(elem, a, (hipStream_t)stream);
    case KV_F16: return load_t<KV_F16>(elem, a, (hipStream_t)stream);
    case KV_E4M3: return load_t<KV_E4M3>(elem, a, (hipStream_t)stream);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
