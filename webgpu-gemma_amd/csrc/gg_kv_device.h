// gg_kv_device.h -- what the kernels on K/V pages share: the sequence of a row
// and the place of a position.
#pragma once
#include "gg_device.h"

namespace gg {

// The last of lo[0, n) that is at most x in an ascending device array (-1: none).
// One wave, 64 probes a time: one load deep up to 64 entries, two up to 4096.
template <class F>
__device__ __forceinline__ int last_at_most(int n, F at_most) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = n;
  while (true) {
    const int step = (span + 63) / 64;
    const int i = lo + lane * step;
    const bool yes = lane * step < span && at_most(i);
    const int c = __popcll(__ballot(yes));
    if (c == 0) return lo - 1;   // only at the first level, where lo is 0
    lo += (c - 1) * step;
    span = min(step, span - (c - 1) * step);
    if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
  }
}

// A sequence's rows and length within the host's bounds.
struct KvSeq {
  int first, rows, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, int s) {
  const int r0 = min(max(a.row_start[s], 0), a.n_rows), r1 = min(max(a.row_start[s + 1], 0), a.n_rows);
  return KvSeq{r0, max(r1 - r0, 0), min(max(a.len[s], 0), a.max_len)};
}
// The sequence that the x-th row or slot belongs to, where sequence s begins at
// begin(row_start[s], s), ascending; -1 if none begins at x or before. Up to 64
// sequences their arrays are read in one go, a sequence a lane: a block's first
// loads are a chain, and this is a link less.
template <class F>
__device__ __forceinline__ int kv_find(const KvArgs& a, long long x, F begin, KvSeq* q) {
  if (a.n_seqs <= 64) {
    const int lane = threadIdx.x & 63, i = min(lane, a.n_seqs - 1);
    const int r0 = min(max(a.row_start[i], 0), a.n_rows), r1 = min(max(a.row_start[i + 1], 0), a.n_rows);
    const int len = min(max(a.len[i], 0), a.max_len);
    const int s = __popcll(__ballot(lane < a.n_seqs && begin(r0, i) <= x)) - 1;
    if (s < 0) return -1;
    q->first = __builtin_amdgcn_readlane(r0, s);
    q->rows = max(__builtin_amdgcn_readlane(r1, s) - q->first, 0);
    q->len = __builtin_amdgcn_readlane(len, s);
    return s;
  }
  const int s = last_at_most(a.n_seqs, [&](int i) { return begin(min(max(a.row_start[i], 0), a.n_rows), i) <= x; });
  if (s >= 0) *q = kv_seq(a, s);
  return s;
}
// The page and place of a position in [0, a.places) of sequence s; false if it has none.
struct KvPlace {
  int page, place;
};
__device__ __forceinline__ bool kv_place(const KvArgs& a, int s, int pos, KvPlace* p) {
  const int i = (int)a.page_div((uint32_t)pos);
  p->page = a.table[(long long)s * a.table_ld + i];
  p->place = pos - i * a.page_size;
  return (uint32_t)p->page < (uint32_t)a.n_pages;
}
// The sequence of a row, -1 if it has none.
__device__ __forceinline__ int kv_seq_of(const KvArgs& a, int row, KvSeq* q) {
  const int s = kv_find(a, row, [](int r, int) { return (long long)r; }, q);
  return s >= 0 && row < q->first + q->rows ? s : -1;
}
__device__ __forceinline__ long long kv_offset(const KvArgs& a, KvPlace p, int head) {
  return p.page * a.page_stride + p.place * a.pos_stride + head * a.head_stride;
}
__device__ __forceinline__ long long kv_scale_at(const KvArgs& a, KvPlace p, int head) {
  return ((long long)p.page * a.page_size + p.place) * a.n_kv + head;
}

}  // namespace gg
