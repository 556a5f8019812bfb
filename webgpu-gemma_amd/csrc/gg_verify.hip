// gg_verify.hip -- drafted tokens against the target's logits.
//
// With p = softmax(z / T) of a row and q the softmax(y / T) that its draft d was
// drawn from, d stands with probability min(1, p(d) / q(d)); else the token is
// drawn from max(p - q, 0): p again in all. Without y, q is 1 at d.
//
// Three launches or four. k_verify_stat reads all rows once: each part's maximum, sum
// of e^((z - m) / T) and best logit. The row at which a sequence stops is found by
// every block of k_verify_sums, or where those are many by k_verify_stop, once.
// k_verify_sums sums that row's weights in f64, kVerifyTile logits a block.
// k_verify_draw finds the tile and the token that the draw falls on.
// Measured, 262144 logits: one sequence, 5 rows of f32: 3.8, 8.0 and 7.0 us, each little
// more than its chain of reads and reductions; 48 sequences, 7 rows each of both
// models, bf16: 37.1 us (4.9 TB/s), 9.0, 22.2 (exponentials in f64) and 9.1.
//
// The draw picks among borders that lie closer than f32 tells apart: with f32
// sums one draw in a hundred over 262144 logits gives a neighbour of the
// right token. So all that a draw compares is f64. So is whether a draft stands: the
// sums of the first launch say so but where u q(d) and p(d) lie closer than they
// can be off (VerifyArgs::near, some 2^-18 of p(d)), and there, at one draft in 10^5,
// both sums are taken again in f64 (0.4 ms for rows of 262144).
// Whether p exceeds q at a token is taken from
// the sums of the first launch: that changes the sum over them in the
// second order only, and their scale is put right afterwards, since
// sum (p - q) over a set = sum p - c sum q with any c. Tiles with a token that the exact c
// puts on the other side are taken again by k_verify_draw, 2 us each (all of them with a draft
// model next to the target: 0.15 ms for rows of 262144).
#include "gg_kv_device.h"

namespace gg {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint64_t logit_key(float z, int i) {
  const uint32_t b = __float_as_uint(z + 0.0f);   // -0 counts as 0
  return ((uint64_t)(b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u)) << 32) | (0xffffffffu - (uint32_t)i);
}
// Wave reductions of 64-bit values on the DPP network, a few cycles a step where
// shuffles through LDS take over a hundred: lanes without a source read 0.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint64_t dpp64(uint64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return ((uint64_t)hi << 32) | lo;
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double x) {
  return __builtin_bit_cast(double, dpp64<CTRL, ROWS>(__builtin_bit_cast(uint64_t, x)));
}
__device__ __forceinline__ uint64_t lane63(uint64_t x) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// Inclusive sums in lane order: within rows of 16, then rows 0 and 2 into the next one, then the first two into the others.
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp_f64<0x111>(x);
  x += dpp_f64<0x112>(x);
  x += dpp_f64<0x114>(x);
  x += dpp_f64<0x118>(x);
  x += dpp_f64<0x142, 0xa>(x);
  x += dpp_f64<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double wave_sum(double x) { return __builtin_bit_cast(double, lane63(__builtin_bit_cast(uint64_t, wave_scan(x)))); }
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
  const auto up = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
  x = up(x, dpp64<0x111>(x));
  x = up(x, dpp64<0x112>(x));
  x = up(x, dpp64<0x114>(x));
  x = up(x, dpp64<0x118>(x));
  x = up(x, dpp64<0x142, 0xa>(x));
  x = up(x, dpp64<0x143, 0xc>(x));
  return lane63(x);
}
__device__ __forceinline__ float wave_top(float x) {
  x = fmaxf(x, dpp_mov_ninf<0x111, 0xf>(x));
  x = fmaxf(x, dpp_mov_ninf<0x112, 0xf>(x));
  x = fmaxf(x, dpp_mov_ninf<0x114, 0xf>(x));
  x = fmaxf(x, dpp_mov_ninf<0x118, 0xf>(x));
  x = fmaxf(x, dpp_mov_ninf<0x142, 0xa>(x));
  x = fmaxf(x, dpp_mov_ninf<0x143, 0xc>(x));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// 2^x for x of 0 or less, f64: 2^round(x) times the Taylor sum of e^r to r^11,
// |r| <= ln(2) / 2, so that 0.347^12 / 12! = 6e-15 of it is left out; under 2^-1100
// it is 0. Under half the instructions of exp(), which is what k_verify_sums is bound by
// (two rows of 262144 for each of 48 sequences).
__device__ __forceinline__ double exp2_below(double x) {
  x = fmax(x, -1100.0);
  const double n = rint(x), r = (x - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800;
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}
constexpr double kLog2e64 = 1.44269504088896340736;

// Temperature of a sequence; 0 (or what is none): greedy. Below 2^-126 its inverse
// is no f32 number.
__device__ __forceinline__ bool greedy(float t) { return !(t > 0.f); }
__device__ __forceinline__ float heat_of(float t) { return greedy(t) ? 1.f : fmaxf(t, 0x1p-126f); }

// One block: part blockIdx % parts of a row of z, or of y behind all of z's.
template <class T, int EPT>
__global__ __launch_bounds__(256) void k_verify_stat(VerifyArgs a) {
  constexpr int VE = 16 / sizeof(T), NV = EPT / VE;
  const int tid = threadIdx.x, lane = tid & 63;
  const long long at = a.block0 + blockIdx.x;
  long long row = at / a.parts;
  const int part = (int)(at - row * a.parts);
  const bool draft = row >= a.rows;
  if (draft) row -= a.rows;
  const int s = last_at_most(a.n_seqs, [&](int i) { return a.row_start[i] <= row; });
  if (s < 0) return;
  const int end = a.row_start[s + 1];
  const float t = a.temperature[s];
  if (row >= end || (draft && (row == end - 1 || greedy(t)))) return;   // no row of y
  // exponents (z - m) log2(e) / T as (z h - m h) c: from T = 2^64 on h keeps the
  // difference of large logits, and c, in range (infinite T: 2^-126, which makes
  // every finite logit's weight 1 and leaves -inf what it is)
  const float heat = heat_of(t), h = heat >= 0x1p64f ? 0x1p-64f : 1.f, c = fmaxf(kLog2e / (heat * h), 0x1p-126f);
  const T* z = draft ? (const T*)a.y + row * a.ldy : (const T*)a.z + row * a.ldz;
  const int shift = (int)(((uintptr_t)z & 15) / sizeof(T));
  const T* z0 = z - shift;
  typedef T vec_t __attribute__((ext_vector_type(VE)));
  float v[EPT];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const long long e0 = ((long long)part * 256 * NV + i * 256 + tid) * VE - shift;
    if (e0 >= 0 && e0 + VE <= a.n) {
      const vec_t x = __builtin_nontemporal_load((const vec_t*)(z + e0));
#pragma unroll
      for (int e = 0; e < VE; ++e) v[i * VE + e] = (float)x[e];
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) v[i * VE + e] = e0 + e >= 0 && e0 + e < a.n ? (float)z[e0 + e] : -INFINITY;
    }
  }
  float m = -INFINITY;
  uint64_t best = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    bad |= !(v[i] < INFINITY);
    m = fmaxf(m, v[i]);
  }
  if (greedy(t)) {
#pragma unroll
    for (int i = EPT - 1; i >= 0; --i)
      if (v[i] == m) best = logit_key(m, (int)(((long long)part * 256 * NV + (i / VE) * 256 + tid) * VE - shift) + i % VE);
    best = wave_max64(best);
  }
  __shared__ float ms[4];
  __shared__ double ss[4];
  __shared__ uint64_t bs[4];
  __shared__ int bads[4];
  const float wm = wave_top(m);
  if (lane == 0) ms[tid >> 6] = wm;
  __syncthreads();
  m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  const float ref = m == -INFINITY ? 0.f : m;
  float sum[4] = {};
#pragma unroll
  for (int i = 0; i < EPT; ++i) sum[i & 3] += __builtin_amdgcn_exp2f(fmaf(v[i], h, -ref * h) * c);
  const double total = wave_sum((double)((sum[0] + sum[1]) + (sum[2] + sum[3])));
  const int any = __ballot(bad) != 0;
  if (lane == 0) {
    ss[tid >> 6] = total;
    bs[tid >> 6] = best;
    bads[tid >> 6] = any;
  }
  __syncthreads();
  if (tid == 0) {
    VerifyPart p;
    p.sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
    p.best = bs[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) p.best = bs[i] > p.best ? bs[i] : p.best;
    p.max = m;
    p.bad = bads[0] | bads[1] | bads[2] | bads[3];
    a.part[at] = p;
  }
}

// A row's parts together, in every lane of a wave.
struct Row {
  float m;
  double sum;
  uint64_t best;
  bool bad;
};
__device__ __forceinline__ Row join_parts(const VerifyPart* p, int n, double c, bool greedy) {
  const int lane = threadIdx.x & 63;
  Row r{-INFINITY, 0.0, 0, false};
  int bad = 0;
  for (int i = lane; i < n; i += 64) {
    r.m = fmaxf(r.m, p[i].max);
    r.best = p[i].best > r.best ? p[i].best : r.best;
    bad |= p[i].bad;
  }
  r.m = wave_top(r.m);
  if (greedy) r.best = wave_max64(r.best);
  for (int i = lane; i < n; i += 64)
    if (p[i].max > -INFINITY) r.sum += p[i].sum * exp2_below(((double)p[i].max - r.m) * c);
  r.sum = wave_sum(r.sum);
  r.bad = __ballot(bad) != 0 || r.m == -INFINITY;
  return r;
}

struct Decision {
  VerifyStop stop;
  int first, end, token;   // token: the one at the stop where none is drawn
  bool greedy;
};

// N logits from e0 on, -inf behind the row.
template <class T, int N>
__device__ __forceinline__ void load_some(const T* row, long long e0, int n, float (&v)[N]) {
  constexpr int VE = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  typedef T vec_t __attribute__((ext_vector_type(VE)));
  if (e0 + N <= n && ((uintptr_t)(row + e0) & (VE * sizeof(T) - 1)) == 0) {
#pragma unroll
    for (int i = 0; i < N; i += VE) {
      const vec_t x = *(const vec_t*)(row + e0 + i);
#pragma unroll
      for (int e = 0; e < VE; ++e) v[i + e] = (float)x[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = e0 + i < n ? (float)row[e0 + i] : -INFINITY;
  }
}
// e^((z - m) / T), c = log2(e) / T. (With an infinite T a logit of -inf gives 0 times
// infinity, a NaN, in whose place exp2_below's fmax takes its bound.)
__device__ __forceinline__ double weight(float z, float m, double c) { return exp2_below(((double)z - (double)m) * c); }

// The sum of a row's weights, every logit's in f64, by a wave.
template <class T>
__device__ __forceinline__ double row_sum(const T* row, int n, float m, double c) {
  const int lane = threadIdx.x & 63;
  double sum = 0;
#pragma unroll 1
  for (long long e0 = 8 * lane; e0 < n; e0 += 512) {
    float z[8];
    load_some(row, e0, n, z);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += weight(z[i], m, c);
  }
  return wave_sum(sum);
}

// Where sequence s stops: four rows at a time, one a wave, up to the first that
// stops. The block with `write` also reports the rows before.
template <class T>
__device__ Decision decide(const VerifyArgs& a, int s, bool write) {
  __shared__ VerifyStop stops[4];
  __shared__ int halts[4], tokens[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  Decision d{};
  d.first = (int)min(max((long long)a.row_start[s], 0ll), a.rows);
  d.end = (int)min(max((long long)a.row_start[s + 1], 0ll), a.rows);
  const float t = a.temperature[s];
  d.greedy = greedy(t);
  const double heat = (double)heat_of(t), c = kLog2e64 / heat;
  d.stop.row = -1;
  for (int r0 = d.first; r0 < d.end; r0 += 4) {
    const int row = r0 + wv;
    if (row < d.end) {
      const bool last = row == d.end - 1;
      Row p = join_parts(a.part + (long long)row * a.parts, a.parts, c, d.greedy);
      const int id = last ? -1 : a.draft[row];
      const bool real = id >= 0 && id < a.n;
      VerifyStop st{row, 0, p.m, 0.f, p.sum, 0.0};
      const int best = (int)(0xffffffffu - (uint32_t)p.best);
      bool halt = last, bad = p.bad;
      int token = best;
      const double z_id = real ? (double)(float)((const T*)a.z)[row * a.ldz + id] : 0.0;
      if (d.greedy) {
        halt |= id != best;
      } else {
        double q = 1.0;
        if (a.y && !last) {
          const Row y = join_parts(a.part + (a.rows + (long long)row) * a.parts, a.parts, c, false);
          bad |= y.bad;
          st.mq = y.m;
          st.sq = y.sum;
          q = real ? exp2_below(((double)(float)((const T*)a.y)[row * a.ldy + id] - y.m) * c) / y.sum : 0.0;
        }
        const double u = real && !last ? a.accept_u[row] : 0.0, w = exp2_below((z_id - p.m) * c);
        bool stands = real && !last && u * q * p.sum < w;
        // closer than f32 exponentials tell: with both sums again
        if (__builtin_expect(real && !last && !bad && w > 0.0 && fabs(u * q * p.sum - w) <= a.near * w, 0)) {
          st.sp = p.sum = row_sum((const T*)a.z + row * a.ldz, a.n, p.m, c);
          if (a.y) {
            q *= st.sq;
            st.sq = row_sum((const T*)a.y + row * a.ldy, a.n, st.mq, c);
            q /= st.sq;
          }
          stands = u * q * p.sum < w;
        }
        halt |= !stands;
        if (halt) st.draw = last ? 1 : a.y ? 3 : 2;
      }
      if (bad) {
        halt = true;
        token = -1;
        st.draw = 0;
      }
      if (lane == 0) {
        stops[wv] = st;
        halts[wv] = halt;
        tokens[wv] = halt ? token : id;
        // whether an earlier wave's row stops is not known yet: what is written here for
        // rows behind the stop is written over below
        if (write) {
          const double z = halt ? (double)p.m : z_id;
          if (a.logprobs) a.logprobs[row] = bad ? NAN : (float)((z - p.m) / heat - log(p.sum));
          a.tokens[row] = halt ? token : id;
        }
      }
    } else if (lane == 0) {
      halts[wv] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 3; i >= 0; --i)
      if (halts[i]) {
        d.stop = stops[i];
        d.token = tokens[i];
      }
    __syncthreads();
    if (d.stop.row >= 0) break;
  }
  return d;
}

// Where sequence s stops; the block with `write` reports it and what lies
// before and behind.
template <class T>
__device__ VerifyStop settle(const VerifyArgs& a, int s, bool write) {
  const int tid = threadIdx.x;
  const Decision d = decide<T>(a, s, write);
  if (write) {
    if (tid == 0) {
      a.accepted[s] = d.stop.row >= 0 ? d.stop.row - d.first : 0;
      a.stop[s] = d.stop;
    }
    if (d.stop.row >= 0)
      for (long long r = d.stop.row + 1ll + tid; r < d.end; r += 256) {
        a.tokens[r] = -1;
        if (a.logprobs) a.logprobs[r] = 0.f;
      }
  }
  return d.stop;
}

template <class T>
__global__ __launch_bounds__(256) void k_verify_stop(VerifyArgs a) {
  settle<T>(a, (int)(a.block0 + blockIdx.x), true);
}

// Block = a tile of a sequence's stop row. With FIND each block finds that row
// for itself, 5 us that a launch of its own takes as well; with many blocks to a
// sequence's tiles and more of them than the CUs hold it has one
// (48 sequences of 262144 logits: 34 us with FIND, 9 and 22 without).
template <class T, bool FIND>
__global__ __launch_bounds__(256) void k_verify_sums(VerifyArgs a) {
  const int tid = threadIdx.x, lane = tid & 63;
  const long long at = a.block0 + blockIdx.x;
  const int s = (int)(at / a.tiles), tile = (int)(at - (long long)s * a.tiles);
  VerifyStop st;
  if constexpr (FIND) st = settle<T>(a, s, tile == 0);
  else st = a.stop[s];
  if (st.row < 0 || st.draw == 0) return;
  const double inv_heat = kLog2e64 / (double)heat_of(a.temperature[s]);
  const long long e0 = (long long)tile * kVerifyTile + 16 * tid;
  const bool both = st.draw == 3;
  const int skip = st.draw == 2 ? a.draft[st.row] : -1;
  double sum[kVerifySums - 1] = {}, border = 1.0;
  // two numbers no further apart than a.near have upper halves, 20 bits of the
  // mantissa, no further apart than this
  const uint32_t near = (uint32_t)(a.near * (1 << 21)) + 2;
  if (e0 < a.n) {
    float z[16], y[16];
    load_some((const T*)a.z + st.row * a.ldz, e0, a.n, z);
    if (both) load_some((const T*)a.y + st.row * a.ldy, e0, a.n, y);
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const double p = weight(z[i], st.mp, inv_heat);
      sum[2] += p;
      if (both) {
        const double q = weight(y[i], st.mq, inv_heat);
        sum[3] += q;
        const double ps = p * st.sq, qs = q * st.sp;
        if (ps > qs) {
          sum[0] += p;
          sum[1] += q;
        }
        // (0 / 0, where both are 0, is passed over by fmin)
        if ((uint32_t)(__double2hiint(ps) - __double2hiint(qs) + near) <= 2 * near) border = fmin(border, fabs(ps - qs) / ps);
      } else if (e0 + i != skip) {
        sum[0] += p;
      }
    }
  }
  __shared__ double part[4][kVerifySums];
#pragma unroll
  for (int k = 0; k < kVerifySums - 1; ++k) {
    if (k % 2 == 1 && !both) continue;   // no q
    const double x = wave_sum(sum[k]);
    if (lane == 0) part[tid >> 6][k] = x;
  }
  // positive f64 numbers are in the order of their bits
  const double least = __ballot(border < 1.0) == 0 ? 1.0 : __builtin_bit_cast(double, ~wave_max64(~__builtin_bit_cast(uint64_t, border)));
  if (lane == 0) part[tid >> 6][kVerifySums - 1] = least;
  __syncthreads();
  if (tid < kVerifySums - 1 && (both || tid % 2 == 0)) a.sums[at * kVerifySums + tid] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
  if (tid == kVerifySums - 1) a.sums[at * kVerifySums + tid] = fmin(fmin(part[0][tid], part[1][tid]), fmin(part[2][tid], part[3][tid]));
}

constexpr int kDrawThreads = 1024, kDrawWaves = kDrawThreads / 64, kDrawEach = kVerifyTile / kDrawThreads;

// Inclusive sums over the block's threads in order.
__device__ double block_scan(double v, double* sh, double* total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const double x = wave_scan(v);
  __syncthreads();
  if (lane == 63) sh[wv] = x;
  __syncthreads();
  double before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kDrawWaves; ++i) {
    before += i < wv ? sh[i] : 0.0;
    all += sh[i];
  }
  *total = all;
  return before + x;
}
// Sums of N values over the block, in every thread. sh: N * kDrawWaves.
template <int N>
__device__ void block_sums(double (&x)[N], double* sh) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const double t = wave_sum(x[k]);
    if (lane == 0) sh[k * kDrawWaves + wv] = t;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    x[k] = 0;
#pragma unroll
    for (int i = 0; i < kDrawWaves; ++i) x[k] += sh[k * kDrawWaves + i];
  }
}

// One block per sequence: the token that the draw falls on.
template <class T>
__global__ __launch_bounds__(kDrawThreads) void k_verify_draw(VerifyArgs a, int seq0) {
  __shared__ double sh[2 * kDrawWaves];
  __shared__ int hit, last, last_p;
  __shared__ double rest;
  const int tid = threadIdx.x, s = seq0 + blockIdx.x;
  const VerifyStop st = a.stop[s];
  if (st.row < 0 || st.draw == 0) return;
  double* sums = a.sums + (long long)s * a.tiles * kVerifySums;
  const double inv_heat = kLog2e64 / (double)heat_of(a.temperature[s]);
  const int per = (a.tiles + kDrawThreads - 1) / kDrawThreads, t0 = min(tid * per, a.tiles), t1 = min(t0 + per, a.tiles);
  // the sums of all p and q first: their quotient scales q
  const bool both = st.draw == 3;
  double p_all = 0, totals[2] = {}, c = 0;
  for (int t = t0; t < t1; ++t) {
    p_all += sums[kVerifySums * t + 2];
    if (both) totals[1] += sums[kVerifySums * t + 3];
  }
  totals[0] = p_all;
  block_sums(totals, sh);
  const double p_sum = totals[0];
  if (both) {
    c = p_sum / totals[1];
    // tokens with p / q between the first launch's quotient and c are on the wrong
    // side: tiles with one that near are summed again
    const double off = 1.0001 * fabs(c * st.sq - st.sp) + 0x1p-45 * st.sp;   // relative to sp; roundings, c for sp / sq
    bool again = false;
    for (int t = t0; t < t1; ++t) again |= sums[kVerifySums * t + 4] * st.sp <= off;
    if (__syncthreads_or(again)) {
      for (int t = 0; t < a.tiles; ++t) {
        if (!(sums[kVerifySums * t + 4] * st.sp <= off)) continue;
        const long long e0 = (long long)t * kVerifyTile + kDrawEach * tid;
        float z[kDrawEach], y[kDrawEach];
        load_some((const T*)a.z + st.row * a.ldz, e0, a.n, z);
        load_some((const T*)a.y + st.row * a.ldy, e0, a.n, y);
        double w[1] = {};
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kDrawEach; ++i) w[0] += fmax(weight(z[i], st.mp, inv_heat) - c * weight(y[i], st.mq, inv_heat), 0.0);
        block_sums(w, sh);
        if (tid == 0) {
          sums[kVerifySums * t] = w[0];
          sums[kVerifySums * t + 1] = 0;
        }
      }
      __syncthreads();
    }
  }
  double mine = 0, all;
  auto tile_weight = [&](int t) { return both ? fmax(sums[kVerifySums * t] - c * sums[kVerifySums * t + 1], 0.0) : sums[kVerifySums * t]; };
  for (int t = t0; t < t1; ++t) mine += tile_weight(t);
  double up_to = block_scan(mine, sh, &all);
  const bool plain = st.draw == 1 || !(all > 0.0);   // nothing left: from p
  if (plain) {
    mine = p_all;
    up_to = block_scan(mine, sh, &all);
  }
  const double target = a.draw_u[s] * all;
  if (tid == 0) {
    hit = a.tiles;
    last = -1;
  }
  __syncthreads();
  {
    // the first tile whose sums pass the target, and the last with any weight
    double x = up_to - mine;
    int first = a.tiles, some = -1;
    double before = 0;
    for (int t = t0; t < t1; ++t) {
      const double w = plain ? sums[kVerifySums * t + 2] : tile_weight(t);
      if (w > 0) some = t;
      if (first == a.tiles && w > 0 && x + w > target) {
        first = t;
        before = x;
      }
      x += w;
    }
    // the threads are in order: a wave's first hit, its last weight
    const uint64_t hits = __ballot(first < a.tiles), any = __ballot(some >= 0);
    if (hits && (tid & 63) == __builtin_ctzll(hits)) atomicMin(&hit, first);
    if (any && (tid & 63) == 63 - __builtin_clzll(any)) atomicMax(&last, some);
    __syncthreads();
    if (first < a.tiles && first == hit) rest = target - before;
    if (hit == a.tiles && tid == 0) rest = INFINITY;   // rounding left none: the last weight
    __syncthreads();
  }
  const int tile = hit < a.tiles ? hit : max(last, 0);
  const double within = rest;
  const long long e0 = (long long)tile * kVerifyTile + kDrawEach * tid;
  const int skip = st.draw == 2 && !plain ? a.draft[st.row] : -1;
  double w[kDrawEach];
  mine = 0;
  int some_p = -1;   // the last id that p has any of
  {
    float z[kDrawEach], y[kDrawEach];
    load_some((const T*)a.z + st.row * a.ldz, e0, a.n, z);
    if (both && !plain) load_some((const T*)a.y + st.row * a.ldy, e0, a.n, y);
#pragma unroll
    for (int i = 0; i < kDrawEach; ++i) {
      w[i] = weight(z[i], st.mp, inv_heat);
      if (w[i] > 0) some_p = (int)(e0 + i);
      if (both && !plain) w[i] = fmax(w[i] - c * weight(y[i], st.mq, inv_heat), 0.0);
      if (e0 + i == skip || e0 + i >= a.n) w[i] = 0;
      mine += w[i];
    }
  }
  __syncthreads();
  up_to = block_scan(mine, sh, &all);
  if (tid == 0) {
    hit = 0x7fffffff;
    last = last_p = -1;
  }
  __syncthreads();
  double x = up_to - mine;
  int first = 0x7fffffff, some = -1;
#pragma unroll
  for (int i = 0; i < kDrawEach; ++i) {
    if (w[i] > 0) some = (int)(e0 + i);
    x += w[i];
    if (first == 0x7fffffff && w[i] > 0 && x > within) first = (int)(e0 + i);
  }
  {
    const uint64_t hits = __ballot(first != 0x7fffffff), any = __ballot(some >= 0);
    if (hits && (tid & 63) == __builtin_ctzll(hits)) atomicMin(&hit, first);
    if (any && (tid & 63) == 63 - __builtin_clzll(any)) atomicMax(&last, some);
  }
  __syncthreads();
  if (__builtin_expect(hit == 0x7fffffff && last < 0, 0)) {
    // the tile's weight was the rounding of p - c q over tokens that have none: the last one that p has any of
    if (some_p >= 0) atomicMax(&last_p, some_p);
    __syncthreads();
  }
  if (tid == 0) {
    const int token = hit != 0x7fffffff ? hit : last >= 0 ? last : max(last_p, 0);
    a.tokens[st.row] = token;
    if (a.logprobs)
      a.logprobs[st.row] = (float)(((double)(float)((const T*)a.z)[st.row * a.ldz + token] - (double)st.mp) / (double)heat_of(a.temperature[s]) - log(p_sum));
  }
}

template <class T>
int verify_t(VerifyArgs a, hipStream_t s) {
  constexpr long long MOST = (1 << 24) - 1;   // a grid holds fewer than 2^32 threads
  const bool few = verify_short(a.rows, a.n);
  const long long stats = (a.y ? 2 : 1) * a.rows * a.parts;
  for (a.block0 = 0; a.block0 < stats; a.block0 += MOST) {
    const unsigned n = (unsigned)(stats - a.block0 < MOST ? stats - a.block0 : MOST);
    if (few) hipLaunchKernelGGL((k_verify_stat<T, kVerifyShort>), dim3(n), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_verify_stat<T, kVerifyLong>), dim3(n), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  const long long sums = (long long)a.n_seqs * a.tiles;
  const bool find = sums <= 1024;
  if (!find) {
    a.block0 = 0;
    hipLaunchKernelGGL((k_verify_stop<T>), dim3((unsigned)a.n_seqs), dim3(256), 0, s, a);   // at most 2^22 blocks
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  for (a.block0 = 0; a.block0 < sums; a.block0 += MOST) {
    const unsigned n = (unsigned)(sums - a.block0 < MOST ? sums - a.block0 : MOST);
    if (find) hipLaunchKernelGGL((k_verify_sums<T, true>), dim3(n), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_verify_sums<T, false>), dim3(n), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  constexpr int DRAWS = 1 << 21;
  for (int at = 0; at < a.n_seqs; at += DRAWS) {
    hipLaunchKernelGGL((k_verify_draw<T>), dim3((unsigned)(a.n_seqs - at < DRAWS ? a.n_seqs - at : DRAWS)), dim3(kDrawThreads), 0, s, a, at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

}  // namespace

int launch_verify(int elem, const VerifyArgs& a, void* stream) {
  switch (elem) {
    case ELEM_F32: return verify_t<float>(a, (hipStream_t)stream);
    case ELEM_F16: return verify_t<_Float16>(a, (hipStream_t)stream);
    case ELEM_BF16: return verify_t<__bf16>(a, (hipStream_t)stream);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace gg
