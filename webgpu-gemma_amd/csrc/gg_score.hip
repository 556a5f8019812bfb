// gg_score.hip -- log probabilities over rows of logits: log-sum-exp, entropy,
// the log probabilities of given ids and the best alternatives.
//
// For a row z of n logits, with m = max z and S = sum e^(z - m):
//   lse = m + ln S,  lp(i) = z_i - lse,
//   entropy = ln S - (sum e^(z - m) (z - m)) / S.
// One pass reads the row once and keeps, per thread, (m, S, W = sum e^(z-m) (z-m))
// relative to the thread's own running maximum:
//   m' = max(m, tile):  W' = e^(m-m') (W + (m - m') S), S' = e^(m-m') S,
// so that partial results of any split merge the same way. All sums are f32.
// Bound by the read of the logits.
//
// Best alternatives: a candidate is a 64-bit key, the logit as an ordered
// integer over the complemented index, so that the largest key is the largest
// logit with the lowest index among equals, and keys differ. A block collects
// in LDS the elements above a threshold that is at most the n-th best so far;
// the first tile's is the n-th largest of the 256 threads' maxima. In index
// order few elements pass later ones (about top ln(n / tile) a row for logits
// in random order); a tile that would overflow the buffer (ties, ascending
// rows) is merged by repeated selection instead, whose cost is bounded.
#include "gg_device.h"

namespace gg {

namespace {

constexpr int kScoreThreads = 256;
constexpr int kScoreBuf = 512;       // candidates a block holds
constexpr int kScoreCompact = 256;   // above this many they are cut to the best `top`

__device__ __forceinline__ uint32_t order_bits(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);   // -0 counts as 0
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t score_key(float z, int i) {
  return ((uint64_t)order_bits(z) << 32) | (0xffffffffu - (uint32_t)i);
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}

struct Stat {
  float m, s, w;
};
// The statistic relative to m >= a.m. The distance is cut at -1e4, where e^d is
// 0 already: d times S stays finite next to masks of the type's lowest value,
// and the empty statistic (m = -inf, S = 0) stays empty.
__device__ __forceinline__ void stat_move(Stat& a, float m) {
  const float d = a.m == m ? 0.f : fmaxf(a.m - m, -1e4f);
  const float f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
  a.w = f * (a.w + d * a.s);
  a.s = f * a.s;
  a.m = m;
}
__device__ __forceinline__ Stat stat_merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  stat_move(a, m);
  stat_move(b, m);
  return Stat{m, a.s + b.s, a.w + b.w};
}
__device__ __forceinline__ Stat stat_shfl(const Stat& a, int o) {
  return Stat{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.w, o, 64)};
}

struct ScoreShared {
  uint64_t buf[kScoreBuf];
  uint64_t list[kScoreMaxTop];
  float mx[kScoreThreads];
  uint64_t wbest[4];
  Stat ws[4];
  float thr;
  int count, add;
};

// The block's merged statistic, in every thread.
__device__ Stat block_stat(ScoreShared& sh, Stat a) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = stat_merge(a, stat_shfl(a, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.ws[threadIdx.x >> 6] = a;
  __syncthreads();
  return stat_merge(stat_merge(sh.ws[0], sh.ws[1]), stat_merge(sh.ws[2], sh.ws[3]));
}

// Largest key of the block below `last` given each thread's, in every thread.
__device__ uint64_t block_best(ScoreShared& sh, uint64_t mine) {
  mine = wave_max64(mine);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wbest[threadIdx.x >> 6] = mine;
  __syncthreads();
  const uint64_t a = sh.wbest[0] > sh.wbest[1] ? sh.wbest[0] : sh.wbest[1];
  const uint64_t b = sh.wbest[2] > sh.wbest[3] ? sh.wbest[2] : sh.wbest[3];
  return a > b ? a : b;
}

// The threshold that `top` of the threads' maxima reach (-inf when fewer than
// `top` have one): at least `top` elements are as large.
__device__ float thread_threshold(ScoreShared& sh, float mx, int top) {
  const int tid = threadIdx.x;
  sh.mx[tid] = mx;
  __syncthreads();
  int rank = 0;
  const float4* p = (const float4*)sh.mx;
#pragma unroll 8
  for (int j = 0; j < kScoreThreads / 4; ++j) {
    const float4 o = p[j];
    rank += (o.x > mx) | ((o.x == mx) & (4 * j < tid));
    rank += (o.y > mx) | ((o.y == mx) & (4 * j + 1 < tid));
    rank += (o.z > mx) | ((o.z == mx) & (4 * j + 2 < tid));
    rank += (o.w > mx) | ((o.w == mx) & (4 * j + 3 < tid));
  }
  if (rank == top - 1) sh.thr = mx;
  __syncthreads();
  return sh.thr;
}

// buf[0, count) -> its best `top` keys in descending order at buf[0, ...);
// returns how many. Every thread calls it; count <= kScoreBuf.
__device__ int compact(ScoreShared& sh, int count, int top) {
  const int tid = threadIdx.x;
  __syncthreads();
  uint64_t k[kScoreBuf / kScoreThreads];
  int rank[kScoreBuf / kScoreThreads] = {};
#pragma unroll
  for (int i = 0; i < kScoreBuf / kScoreThreads; ++i) k[i] = tid + kScoreThreads * i < count ? sh.buf[tid + kScoreThreads * i] : 0;
  for (int j = 0; j < count; ++j) {
    const uint64_t o = sh.buf[j];
#pragma unroll
    for (int i = 0; i < kScoreBuf / kScoreThreads; ++i) rank[i] += o > k[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kScoreBuf / kScoreThreads; ++i)
    if (tid + kScoreThreads * i < count && rank[i] < top) sh.buf[rank[i]] = k[i];
  const int left = count < top ? count : top;
  if (tid == 0) sh.count = left;
  __syncthreads();
  return left;
}

// What the host API reports of a row: the statistic, the given ids' log
// probabilities, and the list buf[0, count).
template <class T>
__device__ void write_row(const ScoreArgs& a, long long row, const Stat& st, const uint64_t* best, int count) {
  const int tid = threadIdx.x;
  const T* z = (const T*)a.z + row * a.ld;
  const float log_s = logf(st.s);
  const bool none = st.s == 0.f;   // every logit is -inf: nothing has a probability
  if (tid == 0) {
    if (a.lse) a.lse[row] = none ? -INFINITY : st.m + log_s;
    if (a.entropy) a.entropy[row] = none ? 0.f : log_s - st.w / st.s;
  }
  for (int j = tid; j < a.n_ids; j += kScoreThreads) {
    const int id = a.ids[row * a.n_ids + j];
    float v = 0.f;   // -1: no token here
    if (id >= 0 && id < a.n) v = none ? -INFINITY : ((float)z[id] - st.m) - log_s;
    else if (id != -1) v = NAN;
    a.lp[row * a.n_ids + j] = v;
  }
  for (int j = tid; j < a.top; j += kScoreThreads) {
    const uint64_t k = j < count ? best[j] : 0;
    if (a.top_ids) a.top_ids[row * a.top + j] = k ? (int)(0xffffffffu - (uint32_t)k) : -1;
    if (a.top_lp) a.top_lp[row * a.top + j] = k ? (order_value((uint32_t)(k >> 32)) - st.m) - log_s : -INFINITY;
  }
}

// One block: chunk blockIdx.x % nch of row blockIdx.x / nch. The row is taken
// in 16-byte units of its address; the units at its ends, which may hold
// elements of other rows, are read element by element.
template <class T, int EPT>
__global__ __launch_bounds__(kScoreThreads) void k_score(ScoreArgs a) {
  constexpr int VE = 16 / sizeof(T), NV = EPT / VE;
  __shared__ ScoreShared sh;
  const int tid = threadIdx.x, top = a.top, n = a.n;
  const long long row = blockIdx.x / a.nch;
  const int ch = blockIdx.x - (int)(row * a.nch);
  const T* z = (const T*)a.z + row * a.ld;
  const int shift = (int)(((uintptr_t)z & 15) / sizeof(T));   // elements of the first unit before the row
  const T* z0 = z - shift;
  const int units = (int)(((long long)n + shift + VE - 1) / VE);
  const int u_lo = ch * a.per, u_hi = min(units, u_lo + a.per);
  if (tid == 0) {
    sh.count = 0;
    sh.add = 0;
  }
  typedef T vec_t __attribute__((ext_vector_type(VE)));
  vec_t nx[NV];
  auto load = [&](int u0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = u0 + i * kScoreThreads + tid;
      const long long e0 = (long long)u * VE - shift;
      if (u < u_hi && e0 >= 0 && e0 + VE <= n) {
        nx[i] = __builtin_nontemporal_load((const vec_t*)z0 + u);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) nx[i][e] = u < u_hi && e0 + e >= 0 && e0 + e < n ? z[e0 + e] : (T)-INFINITY;
      }
    }
  };
  Stat st{-INFINITY, 0.f, 0.f};
  float thr = -INFINITY;
  int count = 0;
  load(u_lo);
  __syncthreads();
  for (int u0 = u_lo; u0 < u_hi; u0 += NV * kScoreThreads) {
    float v[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) v[i * VE + e] = (float)nx[i][e];
    if (u0 + NV * kScoreThreads < u_hi) load(u0 + NV * kScoreThreads);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < EPT; ++i) mx = fmaxf(mx, v[i]);
    mx = fmaxf(mx, -INFINITY);   // all NaN: no maximum
    const float m = fmaxf(st.m, mx);
    stat_move(st, m);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float d = v[i] - ref;
      const float p = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      s += p;
      w = fmaf(p, fmaxf(d, -1e4f), w);   // e^-1e4 is 0: no 0 times -inf
    }
    st.s += s;
    st.w += w;
    if (top > 0) {
      const bool first = thr == -INFINITY;
      float lim = thr;
      if (first) lim = thread_threshold(sh, mx, top);
      auto index = [&](int i) { return (u0 + (i / VE) * kScoreThreads + tid) * VE + i % VE - shift; };
      auto passes = [&](float x) { return first ? (x >= lim) & (x > -INFINITY) : x > lim; };
      int mine = 0;
      if (first ? mx >= lim : mx > lim) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) mine += passes(v[i]) ? 1 : 0;
      }
      int at = 0;
      if (mine) at = atomicAdd(&sh.add, mine);
      __syncthreads();
      const int add = sh.add;
      if (count + add <= kScoreBuf) {
        if (mine) {
          at += count;
#pragma unroll
          for (int i = 0; i < EPT; ++i)
            if (passes(v[i])) sh.buf[at++] = score_key(v[i], index(i));
        }
        count += add;
        if (add && (first || count > kScoreCompact)) {
          count = compact(sh, count, top);
          if (count == top) thr = order_value((uint32_t)(sh.buf[top - 1] >> 32));
        }
      } else {
        // the best `top` of buffer and tile, one by one
        uint64_t last = ~0ull;
        int j = 0;
        for (; j < top; ++j) {
          uint64_t b = 0;
          for (int q = tid; q < count; q += kScoreThreads) {
            const uint64_t k = sh.buf[q];
            b = k < last && k > b ? k : b;
          }
#pragma unroll
          for (int i = 0; i < EPT; ++i) {
            const uint64_t k = passes(v[i]) ? score_key(v[i], index(i)) : 0;
            b = k < last && k > b ? k : b;
          }
          b = block_best(sh, b);
          if (b == 0) break;
          last = b;
          if (tid == 0) sh.list[j] = b;
        }
        __syncthreads();
        if (tid < j) sh.buf[tid] = sh.list[tid];
        count = j;
        __syncthreads();
        if (count == top) thr = order_value((uint32_t)(sh.buf[top - 1] >> 32));
      }
      __syncthreads();
      if (tid == 0) sh.add = 0;
      __syncthreads();
    }
  }
  st = block_stat(sh, st);
  if (top > 0) count = compact(sh, count, top);
  if (a.nch == 1) {
    write_row<T>(a, row, st, sh.buf, count);
    return;
  }
  if (tid == 0) {
    float* p = a.part + 4 * (size_t)blockIdx.x;
    p[0] = st.m;
    p[1] = st.s;
    p[2] = st.w;
  }
  for (int j = tid; j < top; j += kScoreThreads) a.keys[(size_t)blockIdx.x * top + j] = j < count ? sh.buf[j] : 0;
}

// One block per row: the chunks' statistics and lists.
template <class T>
__global__ __launch_bounds__(kScoreThreads) void k_score_merge(ScoreArgs a) {
  __shared__ ScoreShared sh;
  const int tid = threadIdx.x, top = a.top, nch = a.nch;
  const long long row = blockIdx.x;
  Stat st{-INFINITY, 0.f, 0.f};
  if (tid < nch) {
    const float* p = a.part + 4 * ((size_t)row * nch + tid);
    st = Stat{p[0], p[1], p[2]};
  }
  st = block_stat(sh, st);
  int j = 0;
  if (top > 0) {
    // each list descends: a thread holds the front of its chunk's list, and
    // the best front is taken `top` times
    const uint64_t* list = a.keys + ((size_t)row * nch + (tid < nch ? tid : 0)) * top;
    int at = 0;
    uint64_t front = tid < nch ? list[0] : 0;
    for (; j < top; ++j) {
      const uint64_t b = block_best(sh, front);
      if (b == 0) break;
      if (front == b) front = ++at < top ? list[at] : 0;
      if (tid == 0) sh.buf[j] = b;
    }
    __syncthreads();
  }
  write_row<T>(a, row, st, sh.buf, j);
}

template <class T, int EPT>
int launch_score_t(ScoreArgs a, hipStream_t s) {
  hipLaunchKernelGGL((k_score<T, EPT>), dim3((unsigned)(a.rows * a.nch)), dim3(kScoreThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nch == 1) return (int)e;
  hipLaunchKernelGGL((k_score_merge<T>), dim3((unsigned)a.rows), dim3(kScoreThreads), 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace

int launch_score(int elem, const ScoreArgs& a, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  switch (elem) {
    case ELEM_F32: return launch_score_t<float, 32>(a, s);
    case ELEM_F16: return launch_score_t<_Float16, 32>(a, s);
    case ELEM_BF16: return launch_score_t<__bf16, 32>(a, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
