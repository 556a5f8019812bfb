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
// Bound by the read of the logits: 1021 rows of 262144 bf16 (535 MB) with five
// alternatives take 102 to 106 us in a long run of calls, 5.1 to 5.2 TB/s, and up to
// 125 in the first hundred of one, from box to box. One row of f32 is split over
// 129 blocks (8.0 us) and joined by a second kernel (5.7 us): two chains of latencies,
// for 0.2 us of reading.
//
// Best alternatives: a candidate is a 64-bit key, the logit as an ordered
// integer over the complemented index, so that the largest key is the largest
// logit with the lowest index among equals, and keys differ. Every wave keeps
// its own list in LDS: the elements above a bound that is below the block's
// n-th best so far; the first tiles' is near the n-th largest of a wave's lane
// maxima, the waves' best one. In index order few elements pass later ones (for
// logits in random order about n ln(tiles) in a block), which need no barrier;
// a list that grows is cut to its best n, so that every order of logits fits.
// The lists of a block's waves, and then of a row's blocks, are joined by
// counting each key's rank.
#include "gg_device.h"

namespace gg {

namespace {

constexpr int kScoreThreads = 256, kScoreWaves = kScoreThreads / 64;
constexpr int kScoreBuf = 192;       // candidates a wave holds
constexpr int kScoreMore = 16;       // this many above `top` are cut to `top`
constexpr int kScoreLane = 32;       // elements of a tile in a lane, at most
constexpr int kMergePer = 4;         // keys of a row's blocks in a thread that joins them
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
static_assert(kScoreBuf - kScoreMaxTop >= kScoreLane, "a cut list takes what one lane holds");
// The logit of a key, the same in every lane.
__device__ __forceinline__ float list_value(uint64_t key) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(order_value((uint32_t)(key >> 32)))));
}

struct ScoreShared {
  uint64_t buf[kScoreWaves][kScoreBuf], best[kScoreMaxTop];
  float tile[kScoreWaves][kScoreLane];
  float thr[kScoreWaves];   // bounds: the waves' first ones, then their lists' n-th best
  int counts[kScoreWaves];
  Stat ws[kScoreWaves];
};

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The block's merged statistic, in every thread: all lanes move to the wave's
// maximum, then the sums are added.
__device__ Stat block_stat(Stat* ws, Stat a) {   // of the first kScoreWaves waves
  float m = a.m;
  m = fmaxf(m, dpp_mov<0xB1>(m));
  m = fmaxf(m, dpp_mov<0x4E>(m));
  m = fmaxf(m, dpp_mov<0x141>(m));
  m = across8_max(m);
  stat_move(a, m);
  a.s = wave_sum_dpp(a.s);
  a.w = wave_sum_dpp(a.w);
  if ((threadIdx.x & 63) == 0 && threadIdx.x < kScoreThreads) ws[threadIdx.x >> 6] = a;
  __syncthreads();
  return stat_merge(stat_merge(ws[0], ws[1]), stat_merge(ws[2], ws[3]));
}

// A bound that at least n lanes' maxima reach, next to the n-th largest of them
// (-inf when fewer lanes have one). The last six bits give way to the lane, so
// that the order is strict, and count as zero in the bound.
__device__ float lane_threshold(float mx, int n) {
  const int lane = threadIdx.x & 63;
  const uint32_t u = (order_bits(mx) & ~63u) | (uint32_t)(63 - lane);
  int rank = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)u, j) > u;
  const uint64_t at = __ballot(rank == n - 1);
  const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)u, __builtin_ctzll(at)) & ~63u;
  return o > order_bits(-INFINITY) ? order_value(o) : -INFINITY;
}

// buf[0, count) -> its best n keys in descending order; returns how many.
// One wave; count <= kScoreBuf.
__device__ int compact(uint64_t* buf, int count, int n) {
  constexpr int PER = kScoreBuf / 64;
  const int lane = threadIdx.x & 63;
  wave_fence();
  if (count <= 64) {   // a key a lane: no LDS in the loop
    const uint64_t key = lane < count ? buf[lane] : 0;
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), j) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)key, j);
      r += o > key;
    }
    wave_fence();
    if (lane < count && r < n) buf[r] = key;
    wave_fence();
    return min(count, n);
  }
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

// How many of keys[0, n) are above key; eight reads at a time (the last ones of
// n again past its end, not counted).
__device__ __forceinline__ int keys_above(const uint64_t* keys, int n, uint64_t key) {
  int r = 0;
  for (int j = 0; j < n; j += 8) {
    uint64_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = keys[min(j + i, n - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) r += (j + i < n) & (o[i] > key);
  }
  return r;
}

// The thread's first given id and its logit, asked for before the pass: two
// loads that depend on each other.
struct Given {
  int id;
  float z;
};
template <class T>
__device__ __forceinline__ Given given(const ScoreArgs& a, long long row, int j) {
  Given g{-1, 0.f};
  if (j < a.n_ids) g.id = a.ids[row * a.n_ids + j];
  if (g.id >= 0 && g.id < a.n) g.z = (float)((const T*)a.z)[row * a.ld + g.id];
  return g;
}

// What is reported of a row: the statistic, the given ids' log probabilities,
// and the list best[0, top), 0 where there is none.
template <class T, int THREADS>
__device__ void write_row(const ScoreArgs& a, long long row, const Stat& st, const uint64_t* best, Given g) {
  const int tid = threadIdx.x;
  const float log_s = logf(st.s);
  const bool none = st.s == 0.f;   // every logit is -inf: nothing has a probability
  if (tid == 0) {
    if (a.lse) a.lse[row] = none ? -INFINITY : st.m + log_s;
    if (a.entropy) a.entropy[row] = none ? 0.f : log_s - st.w / st.s;
  }
  for (int j = tid; j < a.n_ids; j += THREADS) {
    if (j != tid) g = given<T>(a, row, j);
    float v = 0.f;   // -1: no token here
    if (g.id >= 0 && g.id < a.n) v = none ? -INFINITY : (g.z - st.m) - log_s;
    else if (g.id != -1) v = NAN;
    a.lp[row * a.n_ids + j] = v;
  }
  for (int j = tid; j < a.top; j += THREADS) {
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
  Given g{-1, 0.f};
  if (a.nch == 1) g = given<T>(a, row, tid);
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
  Stat st{-INFINITY, 0.f, 0.f};
  float lim = -INFINITY;   // elements above it may be among the best
  int count = 0;
  const int u_first = u_lo + wv * 64 * NV;
  load(u_first);   // past the chunk's end: -inf
  // every wave takes part in the first round, with or without a tile
  for (int u0 = u_first; u0 < u_hi || u0 == u_first; u0 += STEP) {
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
    if (u0 == u_first) {
      const float t = lane_threshold(mx, top);
      if (lane == 0) sh.thr[wv] = t;
      __syncthreads();
    }
    // another wave's bound may be a logit behind this tile that loses a tie
#pragma unroll
    for (int q = 0; q < kScoreWaves; ++q) {
      const float t = __hip_atomic_load(&sh.thr[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      lim = fmaxf(lim, t == -INFINITY ? t : before(t));
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
        count = compact(buf, count, top);                        // to `top`: it was full
        lim = fmaxf(lim, before(list_value(buf[top - 1])));      // within the tile the order is not the indices'
        mask = __ballot(x > lim);
      }
      if (x > lim)
        buf[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u))] =
            score_key(x, (u0 + 64 * (lane / VE) + L) * VE + lane % VE - shift);
      count += __popcll(mask);
    }
    if (count >= top + kScoreMore) {
      count = compact(buf, count, top);
      const float t = list_value(buf[top - 1]);
      lim = fmaxf(lim, t);   // all of the list comes before the next tile: it wins ties
      if (lane == 0) __hip_atomic_store(&sh.thr[wv], t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  if (top > 0) {
    if (count > kScoreThreads / kScoreWaves) count = compact(buf, count, top);
    if (lane == 0) sh.counts[wv] = count;
  }
  st = block_stat(sh.ws, st);   // and the waves' lists are complete
  if (top > 0) {
    // a key a thread
    uint64_t key = 0;
    int rank = 0, at = tid;
#pragma unroll
    for (int q = 0; q < kScoreWaves; ++q) {
      const int c = sh.counts[q];
      if (at >= 0 && at < c) key = sh.buf[q][at];
      at -= c;
    }
    if (key) {
      for (int q = 0; q < kScoreWaves; ++q) rank += keys_above(sh.buf[q], sh.counts[q], key);
    }
    if (tid < top) sh.best[tid] = 0;
    __syncthreads();
    if (key && rank < top) sh.best[rank] = key;
    __syncthreads();
  }
  if (a.nch == 1) {
    write_row<T, kScoreThreads>(a, row, st, sh.best, g);
    return;
  }
  if (tid == 0) {
    float* p = a.part + 4 * (size_t)blockIdx.x;
    p[0] = st.m;
    p[1] = st.s;
    p[2] = st.w;
  }
  for (int j = tid; j < top; j += kScoreThreads) a.keys[(size_t)blockIdx.x * top + j] = sh.best[j];
}

// One block per row: the chunks' statistics and lists. At most 4096 keys, four
// a thread; the ranks are counted of those whose logit reaches a bound
// that `top` of 64 groups' best do (about 2 top of them without ties).
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_score_merge(ScoreArgs a) {
  constexpr int PER = kMergePer;
  __shared__ Stat ws[kScoreWaves];
  __shared__ __align__(16) float own[THREADS];
  __shared__ uint64_t cand[THREADS * PER], best[kScoreMaxTop];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, top = a.top, nch = a.nch;
  const long long row = blockIdx.x;
  const int total = nch * top;
  uint64_t k[PER], b = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) k[i] = tid + THREADS * i < total ? a.keys[(size_t)row * total + tid + THREADS * i] : 0;
  Stat st{-INFINITY, 0.f, 0.f};
  if (tid < nch) {
    const float* p = a.part + 4 * ((size_t)row * nch + tid);
    st = Stat{p[0], p[1], p[2]};
  }
  const Given g = given<T>(a, row, tid);
#pragma unroll
  for (int i = 0; i < PER; ++i) b = k[i] > b ? k[i] : b;
  own[tid] = b ? order_value((uint32_t)(b >> 32)) : -INFINITY;
  if (tid < top) best[tid] = 0;
  if (tid == 0) count = 0;
  static_assert(kScoreMaxChunks <= kScoreThreads, "the first waves hold the statistics");
  st = block_stat(ws, st);
  if (top > 0) {
    // every wave finds the bound for itself
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < THREADS / 256; ++i) {
      const float4 o = *(const float4*)&own[256 * i + 4 * lane];
      mx = fmaxf(fmaxf(fmaxf(o.x, o.y), fmaxf(o.z, o.w)), mx);
    }
    const float lim = lane_threshold(mx, top);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool take = k[i] != 0 && order_value((uint32_t)(k[i] >> 32)) >= lim;
      const uint64_t mask = __ballot(take);
      if (!mask) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(&count, (int)__popcll(mask));
      at = __builtin_amdgcn_readfirstlane(at);
      if (take) cand[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u))] = k[i];
    }
    __syncthreads();
    const int c = count;
    for (int i = tid; i < c; i += THREADS) {
      const uint64_t key = cand[i];
      const int r = keys_above(cand, c, key);
      if (r < top) best[r] = key;
    }
    __syncthreads();
  }
  write_row<T, THREADS>(a, row, st, best, g);
}

template <class T, int EPT>
int launch_score_t(ScoreArgs a, hipStream_t s) {
  // a launch for each 2^22 rows: a grid holds fewer than 2^32 threads (more
  // rows than 768 are one block each)
  constexpr long long MOST = 1 << 22;
  for (long long left = a.rows; left > 0; left -= MOST) {
    a.rows = left < MOST ? left : MOST;
    hipLaunchKernelGGL((k_score<T, EPT>), dim3((unsigned)(a.rows * a.nch)), dim3(kScoreThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    if (left <= MOST) break;
    a.z = (const T*)a.z + MOST * a.ld;
    if (a.n_ids) {
      a.ids += MOST * a.n_ids;
      a.lp += MOST * a.n_ids;
    }
    if (a.lse) a.lse += MOST;
    if (a.entropy) a.entropy += MOST;
    if (a.top_ids) a.top_ids += MOST * a.top;
    if (a.top_lp) a.top_lp += MOST * a.top;
  }
  if (a.nch == 1) return 0;
  if (a.nch * a.top <= kScoreThreads * kMergePer)
    hipLaunchKernelGGL((k_score_merge<T, kScoreThreads>), dim3((unsigned)a.rows), dim3(kScoreThreads), 0, s, a);
  else
    hipLaunchKernelGGL((k_score_merge<T, 1024>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace

int launch_score(int elem, const ScoreArgs& a, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  const bool few = a.tile < kScoreTile;
  switch (elem) {
    case ELEM_F32: return few ? launch_score_t<float, 8>(a, s) : launch_score_t<float, 32>(a, s);
    case ELEM_F16: return few ? launch_score_t<_Float16, 8>(a, s) : launch_score_t<_Float16, 32>(a, s);
    case ELEM_BF16: return few ? launch_score_t<__bf16, 8>(a, s) : launch_score_t<__bf16, 32>(a, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
