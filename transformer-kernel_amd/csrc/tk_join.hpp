// Attention whose keys are split over workgroups: what they leave behind, and the launch that joins it.
//
// A row is one query of one head.  Split s of row r leaves, in a slot of its own, its unnormalised
// output O (fp32, hd values) relative to its reference m (weight_ref: in units of log2, a little
// below its largest score), and {m, sum of weights}; a split that saw no key leaves m = -inf and no
// O.  The row is sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s with m the largest m_s, and zeros where
// nothing was seen.
#pragma once
#include "tk_elem.hpp"

namespace tk {
namespace {

struct JoinArgs {
  const float* part;   // [slots][hd]
  const float* stats;  // [slots][2]
  void* o;
  // Nullable: {first slot w, splits} of each sequence.  Split s of a row lies in slot (w + s) * heads + h; one
  // split alone is the output already.  Without a plan row r's splits lie in slots r * splits + s.
  const int32_t* plan;
  int64_t os[3];        // elements, {b, h, s}
  int heads, q_len, hd;
  int splits;  // without a plan: of every row; with one: about how many
  int64_t rows;
};

constexpr int kJoinWaves = 4;

// A result in the making: reference, sum of weights and 4 columns of O relative to the reference.
struct JoinPart {
  float m, l;
  f32x4 o;
  __device__ __forceinline__ void add(float m2, float l2, f32x4 o2) {
    const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
    m = top;
    l = f * l + f2 * l2;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = f * o[e] + f2 * o2[e];
  }
};

// GROUPED: a workgroup joins 16 columns of a row, with 64 groups of 4 lanes; else a wave joins a row, with
// groups of 16, 32 or 64 lanes.  Group i takes splits i, i + groups, ..., and the groups are merged as one
// tree, so the sums have one order whatever the batch.  A chain of load latencies (the plan, the results),
// so nothing waits for the maximum of all splits: 256 splits of 16 rows of 128 take 4.0 us, 2 of 1024 rows
// 4.8 (the same work behind a first pass for the maximum, and summed group by group, 6.6).
template <typename T, bool GROUPED>
__global__ __launch_bounds__(kJoinWaves * 64) void split_join_kernel(JoinArgs p) {
  __shared__ JoinPart lds[GROUPED ? kJoinWaves : 1][4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int blocks = GROUPED ? (p.hd + 15) / 16 : 1;
  const int64_t rowid = GROUPED ? blockIdx.x / blocks : (int64_t)blockIdx.x * kJoinWaves + wave;
  if (rowid >= p.rows) return;
  const int64_t bh = rowid / p.q_len;
  const int b = (int)(bh / p.heads), h = (int)(bh % p.heads);
  const int splits = p.plan ? p.plan[2 * b + 1] : p.splits;
  if (p.plan && splits == 1) return;
  const int64_t base = p.plan ? (int64_t)p.plan[2 * b] * p.heads + h : rowid * p.splits;
  const int64_t step = p.plan ? p.heads : 1;
  const int lpr = GROUPED ? 4 : p.hd <= 64 ? 16 : p.hd <= 128 ? 32 : 64;
  const int groups = (GROUPED ? kJoinWaves * 64 : 64) / lpr, grp = (GROUPED ? (int)threadIdx.x : lane) / lpr;
  const int d = (GROUPED ? (int)(blockIdx.x % blocks) * 16 : 0) + lane % lpr * 4, dc = min(d, p.hd - 4);

  JoinPart r = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int s = grp; s < splits; s += groups) {
    const int64_t at = base + s * step;
    const f32x2 st = *reinterpret_cast<const f32x2*>(p.stats + 2 * at);
    f32x4 o = *reinterpret_cast<const f32x4*>(p.part + at * p.hd + dc);
    if (st[0] == -INFINITY) o = f32x4{0.f, 0.f, 0.f, 0.f};  // an empty split wrote no O
    r.add(st[0], st[1], o);
  }
  for (int off = lpr; off < 64; off <<= 1) {
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __shfl_xor(r.o[e], off);
    r.add(__shfl_xor(r.m, off), __shfl_xor(r.l, off), o);
  }
  if constexpr (GROUPED) {
    if (lane < 4) lds[wave][lane] = r;
    __syncthreads();
    if (threadIdx.x >= 4) return;
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) r.add(lds[w][lane].m, lds[w][lane].l, lds[w][lane].o);
  }
  if (lane >= lpr || d >= p.hd) return;
  T* out = reinterpret_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + rowid % p.q_len * p.os[2] + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(r.l == 0.f ? 0.f : r.o[e] / r.l);
}

// Few splits: a wave per row.  one_order: the tree of the groups, in which splits that a longer table adds
// (empty ones) change no bit.
inline bool join_grouped(int64_t splits, bool one_order) { return one_order || splits > 16; }

// Workgroups of the join; above kMaxGroups the whole call is to be refused, before its first launch.
inline int64_t join_grid(int64_t rows, int64_t hd, int64_t splits, bool one_order) {
  return join_grouped(splits, one_order) ? rows * ((hd + 15) / 16) : (rows + kJoinWaves - 1) / kJoinWaves;
}

template <typename T>
int launch_join(const char* fn, const JoinArgs& p, bool one_order, hipStream_t st) {
  const bool grouped = join_grouped(p.splits, one_order);
  const dim3 g((unsigned)join_grid(p.rows, p.hd, p.splits, one_order)), blk(kJoinWaves * 64);
  if (grouped) hipLaunchKernelGGL((split_join_kernel<T, true>), g, blk, 0, st, p);
  else hipLaunchKernelGGL((split_join_kernel<T, false>), g, blk, 0, st, p);
  return check_launch(fn);
}

}  // namespace
}  // namespace tk
