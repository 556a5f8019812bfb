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
// logit with the lowest index among equals, and keys differ. Every wave keeps
// its own list in LDS, without a barrier in the pass: the elements above a
// threshold that is at most the block's n-th best so far; the first tile's is
// the n-th largest of the lanes' maxima. In index order few elements pass
// later ones (for logits in random order about n ln(tiles) in a block); a full
// list is cut to its best n, so that every order of logits fits. The lists of a
// block's waves, and then of a row's blocks, are joined by counting each key's
// rank.
#include "gg_device.h"

namespace gg {

namespace {

constexpr int kScoreThreads = 256, kScoreWaves = kScoreThreads / 64;
constexpr int kScoreBuf = 192;       // candidates a wave holds
constexpr int kScoreCompact = 128;   // above this many they are cut to the best `top`
constexpr int kScoreLane = 32;       // elements of a tile in a lane, at most
constexpr int kScoreJoin = 4096;     // keys of a row's blocks
static_assert(kScoreWaves * kScoreMaxTop <= kScoreThreads, "a key a thread");

__device__ __forceinline__ uint32_t order_bits(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);   // -0 counts as 0
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
// The next f32 below x (finite or +inf); below 0 it is the one below -0.
__device__ __forceinline__ float before(float x) { return order_value(order_bits(x) - (x == 0.f ? 2u : 1u)); }
__device__ __forceinline__ uint64_t score_key(float z, int i) {
  return ((uint64_t)order_bits(z) << 32) | (0xffffffffu - (uint32_t)i);
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

static_assert(kScoreBuf - kScoreMaxTop >= 64 && kScoreCompact >= kScoreMaxTop, "a cut list takes what one lane holds");
// The logit of a key, the same in every lane.
__device__ __forceinline__ float list_value(uint64_t key) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(order_value((uint32_t)(key >> 32)))));
}

struct ScoreShared {
  uint64_t buf[kScoreWaves][kScoreBuf];
  float mx[kScoreWaves][64];
  float tile[kScoreWaves][kScoreLane];
  float thr[kScoreWaves];   // the waves' thresholds
  Stat ws[kScoreWaves];
};

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The block's merged statistic, in every thread.
__device__ Stat block_stat(Stat* ws, Stat a) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = stat_merge(a, stat_shfl(a, o));
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = a;
  __syncthreads();
  return stat_merge(stat_merge(ws[0], ws[1]), stat_merge(ws[2], ws[3]));
}

// The n-th largest of the lanes' maxima (-inf when fewer lanes have one): at
// least n elements are as large.
__device__ float lane_threshold(float* mxs, float mx, int n) {
  const int lane = threadIdx.x & 63;
  mxs[lane] = mx;
  wave_fence();
  int rank = 0;
  const float4* p = (const float4*)mxs;
#pragma unroll 4
  for (int j = 0; j < 16; ++j) {
    const float4 o = p[j];
    rank += (o.x > mx) | ((o.x == mx) & (4 * j < lane));
    rank += (o.y > mx) | ((o.y == mx) & (4 * j + 1 < lane));
    rank += (o.z > mx) | ((o.z == mx) & (4 * j + 2 < lane));
    rank += (o.w > mx) | ((o.w == mx) & (4 * j + 3 < lane));
  }
  const uint64_t at = __ballot(rank == n - 1);   // the ranks are a permutation
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mx), __builtin_ctzll(at)));
}

// buf[0, count) -> its best n keys in descending order; returns how many.
// One wave; count <= kScoreBuf.
__device__ int compact(uint64_t* buf, int count, int n) {
  constexpr int PER = kScoreBuf / 64;
  const int lane = threadIdx.x & 63;
  wave_fence();
  uint64_t k[PER];
  int rank[PER] = {};
#pragma unroll
  for (int i = 0; i < PER; ++i) k[i] = lane + 64 * i < count ? buf[lane + 64 * i] : 0;
#pragma unroll 4
  for (int j = 0; j < count; ++j) {
    const uint64_t o = buf[j];
#pragma unroll
    for (int i = 0; i < PER; ++i) rank[i] += o > k[i];
  }
  wave_fence();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < count && rank[i] < n) buf[rank[i]] = k[i];
  wave_fence();
  return __builtin_amdgcn_readfirstlane(min(count, n));
}

// What the host API reports of a row: the statistic, the given ids' log
// probabilities, and the list best[0, top), 0 where there is none.
template <class T>
__device__ void write_row(const ScoreArgs& a, long long row, const Stat& st, const uint64_t* best) {
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
    const uint64_t k = best[j];
    if (a.top_ids) a.top_ids[row * a.top + j] = k ? (int)(0xffffffffu - (uint32_t)k) : -1;
    if (a.top_lp) a.top_lp[row * a.top + j] = k ? (order_value((uint32_t)(k >> 32)) - st.m) - log_s : -INFINITY;
  }
}

// One block: chunk blockIdx.x % nch of row blockIdx.x / nch; its waves take
// turns at tiles of 64 EPT elements. The row is taken in 16-byte units of its
// address; the units at its ends, which may hold elements of other rows, are
// read element by element.
template <class T, int EPT>
__global__ __launch_bounds__(kScoreThreads, 4) void k_score(ScoreArgs a) {
  static_assert(EPT <= kScoreLane, "a lane's part of a tile");
  constexpr int VE = 16 / sizeof(T), NV = EPT / VE, STEP = NV * kScoreThreads;
  __shared__ ScoreShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), top = a.top, n = a.n;
  const long long row = blockIdx.x / a.nch;
  const int ch = blockIdx.x - (int)(row * a.nch);
  const T* z = (const T*)a.z + row * a.ld;
  const int shift = (int)(((uintptr_t)z & 15) / sizeof(T));   // elements of the first unit before the row
  const T* z0 = z - shift;
  const int units = (int)(((long long)n + shift + VE - 1) / VE);
  const int u_lo = ch * a.per, u_hi = min(units, u_lo + a.per);
  uint64_t* buf = sh.buf[wv];
  typedef T vec_t __attribute__((ext_vector_type(VE)));
  vec_t nx[NV];
  auto load = [&](int u0) __attribute__((always_inline)) {
    if (u0 * VE >= shift && u0 + 64 * NV <= u_hi && (long long)(u0 + 64 * NV) * VE - shift <= n) {
#pragma unroll
      for (int i = 0; i < NV; ++i) nx[i] = __builtin_nontemporal_load((const vec_t*)z0 + (u0 + i * 64 + lane));
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int u = u0 + i * 64 + lane;
        const long long e0 = (long long)u * VE - shift;
        if (u < u_hi && e0 >= 0 && e0 + VE <= n) {
          nx[i] = __builtin_nontemporal_load((const vec_t*)z0 + u);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) nx[i][e] = u < u_hi && e0 + e >= 0 && e0 + e < n ? z[e0 + e] : (T)-INFINITY;
        }
      }
    }
  };
  if (tid < kScoreWaves) sh.thr[tid] = -INFINITY;
  __syncthreads();
  Stat st{-INFINITY, 0.f, 0.f};
  float thr = -INFINITY;
  int count = 0;
  const int u_first = u_lo + wv * 64 * NV;
  if (u_first < u_hi) load(u_first);
  for (int u0 = u_first; u0 < u_hi; u0 += STEP) {
    float v[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) v[i * VE + e] = (float)nx[i][e];
    if (u0 + STEP < u_hi) load(u0 + STEP);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < EPT; ++i) mx = fmaxf(mx, v[i]);
    mx = fmaxf(mx, -INFINITY);   // all NaN: no maximum
    const float m = fmaxf(st.m, mx);
    if (__ballot(m > st.m)) stat_move(st, m);
    const float ref = m == -INFINITY ? 0.f : m;
    float s[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float d = v[i] - ref;
      const float p = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      s[i & 1] += p;
      w[i & 1] = fmaf(p, fmaxf(d, -1e4f), w[i & 1]);   // e^-1e4 is 0: no 0 times -inf
    }
    st.s += s[0] + s[1];
    st.w += w[0] + w[1];
    if (top == 0) continue;
    // Above `lim` an element may be one of the best: this wave's own n-th best
    // came before the tile and wins a tie, another wave's may not.
    float lim = thr;
#pragma unroll
    for (int q = 0; q < kScoreWaves; ++q) {
      const float t = __hip_atomic_load(&sh.thr[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      lim = q == wv || t == -INFINITY ? lim : fmaxf(lim, before(t));
    }
    const bool first = __builtin_amdgcn_readfirstlane(lim == -INFINITY);
    if (first) {
      const float t = lane_threshold(sh.mx[wv], mx, top);
      lim = t == -INFINITY ? t : before(t);
    }
    uint64_t lanes = __ballot(mx > lim);
    if (lanes == 0) continue;
    if (__popcll(lanes) > 4) {
      // many lanes, as in the first tile: each writes its elements to its place
      int c = 0;
#pragma unroll
      for (int i = 0; i < EPT; ++i) c += v[i] > lim;
      int at = count, sum = 0;
#pragma unroll
      for (int bit = 0; (EPT >> bit) > 0; ++bit) {   // prefix sums, a bit of the counts at a time
        const uint64_t mask = __ballot((c >> bit) & 1);
        at += __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u)) << bit;
        sum += __popcll(mask) << bit;
      }
      if (count + sum <= kScoreBuf) {
        const int e_lane = (u0 + lane) * VE - shift;
#pragma unroll
        for (int i = 0; i < EPT; ++i)
          if (v[i] > lim) buf[at++] = score_key(v[i], e_lane + 64 * VE * (i / VE) + i % VE);
        count += sum;
        lanes = 0;
      }
    }
    // one lane's elements at a time, an element a lane: any number of them fits
    float* tile = sh.tile[wv];
    while (lanes) {
      const int L = __builtin_ctzll(lanes);
      lanes &= lanes - 1;
      if (lane == L) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) tile[i] = v[i];
      }
      wave_fence();
      const float x = lane < EPT ? tile[lane] : -INFINITY;
      wave_fence();
      uint64_t mask = __ballot(x > lim);
      if (count + __popcll(mask) > kScoreBuf) {
        count = compact(buf, count, top);   // to `top`: it was full
        thr = list_value(buf[top - 1]);
        lim = fmaxf(lim, before(thr));      // within the tile the order is not the indices'
        mask = __ballot(x > lim);
      }
      if (x > lim)
        buf[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u))] =
            score_key(x, (u0 + 64 * (lane / VE) + L) * VE + lane % VE - shift);
      count += __popcll(mask);
    }
    if (count > kScoreCompact || (first && count >= top)) {
      count = compact(buf, count, top);
      thr = list_value(buf[top - 1]);
    }
    if (lane == 0) __hip_atomic_store(&sh.thr[wv], thr, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  if (top > 0) {
    count = compact(buf, count, top);
    for (int j = count + lane; j < top; j += 64) buf[j] = 0;
  }
  st = block_stat(sh.ws, st);   // and the waves' lists are complete
  // the waves' lists, a key a thread
  uint64_t key = 0;
  int rank = 0;
  if (top > 0) {
    const int lw = tid / top, lj = tid - lw * top;
    if (lw < kScoreWaves) key = sh.buf[lw][lj];
    for (int q = 0; q < kScoreWaves; ++q)
      for (int j = 0; j < top; ++j) rank += sh.buf[q][j] > key;
    __syncthreads();
    uint64_t* best = sh.buf[0];
    if (tid < top) best[tid] = 0;
    __syncthreads();
    if (key && rank < top) best[rank] = key;
    __syncthreads();
  }
  if (a.nch == 1) {
    write_row<T>(a, row, st, sh.buf[0]);
    return;
  }
  if (tid == 0) {
    float* p = a.part + 4 * (size_t)blockIdx.x;
    p[0] = st.m;
    p[1] = st.s;
    p[2] = st.w;
  }
  for (int j = tid; j < top; j += kScoreThreads) a.keys[(size_t)blockIdx.x * top + j] = sh.buf[0][j];
}

// One block per row: the chunks' statistics and lists. At most kScoreJoin keys,
// 16 a thread; the ranks are counted of those whose logit is at least the
// `top`-th largest of 64 groups' best (about 2 top of them without ties).
template <class T>
__global__ __launch_bounds__(kScoreThreads) void k_score_merge(ScoreArgs a) {
  constexpr int PER = kScoreJoin / kScoreThreads;
  __shared__ Stat ws[kScoreWaves];
  __shared__ __align__(16) float own[kScoreThreads];
  __shared__ uint64_t cand[kScoreJoin], best[kScoreMaxTop];
  __shared__ float limit;
  __shared__ int count;
  const int tid = threadIdx.x, top = a.top, nch = a.nch;
  const long long row = blockIdx.x;
  Stat st{-INFINITY, 0.f, 0.f};
  if (tid < nch) {
    const float* p = a.part + 4 * ((size_t)row * nch + tid);
    st = Stat{p[0], p[1], p[2]};
  }
  const int total = nch * top;
  uint64_t k[PER], b = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) k[i] = tid + kScoreThreads * i < total ? a.keys[(size_t)row * total + tid + kScoreThreads * i] : 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) b = k[i] > b ? k[i] : b;
  own[tid] = b ? order_value((uint32_t)(b >> 32)) : -INFINITY;
  if (tid < top) best[tid] = 0;
  if (tid == 0) count = 0;
  st = block_stat(ws, st);
  if (top > 0) {
    if (tid < 64) {
      const float g = fmaxf(fmaxf(own[tid], own[tid + 64]), fmaxf(own[tid + 128], own[tid + 192]));
      wave_fence();
      const float lim = lane_threshold(own, g, top);
      if (tid == 0) limit = lim;
    }
    __syncthreads();
    const float lim = limit;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (k[i] && order_value((uint32_t)(k[i] >> 32)) >= lim) cand[atomicAdd(&count, 1)] = k[i];
    __syncthreads();
    const int c = count;
    for (int i = tid; i < c; i += kScoreThreads) {
      const uint64_t key = cand[i];
      int r = 0;
#pragma unroll 4
      for (int j = 0; j < c; ++j) r += cand[j] > key;
      if (r < top) best[r] = key;
    }
    __syncthreads();
  }
  write_row<T>(a, row, st, best);
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
