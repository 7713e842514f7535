// Attention whose keys are split over workgroups: what they leave behind, and the launch that joins it.
//
// A row is one query of one head.  Split s of row r leaves its unnormalised output O (fp32, hd
// values) relative to its running maximum m (in units of log2), and {m, sum of weights}; a split
// that saw no key leaves m = -inf and no O.  The row is sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s
// with m the largest m_s, and zeros where nothing was seen.
#pragma once
#include "tk_elem.hpp"

namespace tk {
namespace {

struct JoinArgs {
  const float* part;   // [rows][splits][hd]
  const float* stats;  // [rows][splits][2]
  void* o;
  int64_t os[3];  // elements, {b, h, s}
  int heads, q_len, hd, splits;
  int cols;  // columns of a row that a workgroup joins
};

constexpr int kJoin = 256;

// Workgroups of kJoin / lpr groups of lpr lanes with 4 columns each, group i taking splits i, i + groups,
// ...; the groups are added in their order, so the sums have one order whatever the batch.  (One wave that
// walked 391 splits of a row of 128 alone took 235 us, 16 groups of one workgroup 16 us.)
template <typename T>
__global__ __launch_bounds__(kJoin) void split_join_kernel(JoinArgs p) {
  __shared__ float m_lds[kJoin / 64];
  __shared__ f32x4 o_lds[kJoin];
  __shared__ float l_lds[kJoin];
  const int blocks = (p.hd + p.cols - 1) / p.cols;
  const int64_t rowid = blockIdx.x / blocks;
  const float* st = p.stats + 2 * rowid * p.splits;
  float m = -INFINITY;
  for (int s = threadIdx.x; s < p.splits; s += kJoin) m = fmaxf(m, st[2 * s]);
  m = group_max<64>(m);
  if ((threadIdx.x & 63) == 0) m_lds[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoin / 64; ++w) m = fmaxf(m, m_lds[w]);
  const float m_ref = m == -INFINITY ? 0.f : m;

  const int lpr = p.cols / 4, groups = kJoin / lpr;
  const int grp = threadIdx.x / lpr, d = (int)(blockIdx.x % blocks) * p.cols + (threadIdx.x % lpr) * 4;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  if (d < p.hd) {
    const float* part = p.part + rowid * p.splits * p.hd + d;
#pragma unroll 4
    for (int s = grp; s < p.splits; s += groups) {
      if (st[2 * s] == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(st[2 * s] - m_ref);
      const f32x4 o = *reinterpret_cast<const f32x4*>(part + (int64_t)s * p.hd);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, o[e], sum[e]);
      l = fmaf(f, st[2 * s + 1], l);
    }
  }
  o_lds[threadIdx.x] = sum;
  l_lds[threadIdx.x] = l;
  __syncthreads();
  if (grp != 0 || d >= p.hd) return;
  for (int i = 1; i < min(groups, p.splits); ++i) {
    const f32x4 o = o_lds[i * lpr + threadIdx.x];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += o[e];
    l += l_lds[i * lpr + threadIdx.x];
  }
  const int64_t bh = rowid / p.q_len;
  T* out = reinterpret_cast<T*>(p.o) + bh / p.heads * p.os[0] + bh % p.heads * p.os[1] + rowid % p.q_len * p.os[2] + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(l == 0.f ? 0.f : sum[e] / l);
}

template <typename T>
int launch_join(const char* fn, JoinArgs p, int64_t rows, hipStream_t st) {
  // many splits: 16 columns to a workgroup, so that 64 groups share them; few: a row to a workgroup
  p.cols = p.splits > 32 ? 16 : p.hd <= 64 ? 64 : p.hd <= 128 ? 128 : 256;
  const int64_t grid = rows * ((p.hd + p.cols - 1) / p.cols);
  TK_REQUIRE(grid < (1ll << 31), TK_ERR_UNSUPPORTED, "%s: too many rows", fn);
  hipLaunchKernelGGL((split_join_kernel<T>), dim3((unsigned)grid), dim3(kJoin), 0, st, p);
  return check_launch(fn);
}

}  // namespace
}  // namespace tk
