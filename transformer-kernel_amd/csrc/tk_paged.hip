// Attention of one new token per sequence over a paged key/value cache.
//
//   o[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j   over the keys j of sequence b that
// the token at position lengths[b] - 1 sees: j < lengths[b], and with a window also
// j >= lengths[b] - window or j < sinks.  Key j is row j % page_size of page
// table[b][j / page_size], in every page the rows of one key head together or not (strides).
//
// Bound by the bytes of K and V, each read once: the G = heads / kv_heads query heads that
// share a key head are the columns of one matrix product (up to 16 of them; the unused ones
// are zeros, the matrix cores idle anyway).  Per step a wave takes 32 keys:
//   S^T[key, head] = K . Q^T, two 16x16 tiles; A operand: lane l holds key l & 15, 16 bytes
//     straight from the page, no LDS.
//   softmax over the accumulator: lane l holds head l & 15 and keys 16t + 4g + r (g = l >> 4),
//     so a head's running maximum is two lane exchanges and the rescale one factor per lane.
//   O^T[d, head] += V^T . P^T: the accumulator's keys are taken as the product's k slots as they
//     lie (slot 8g + 4t + r), so P needs no move; lane l loads the CW = DT/16 neighbouring
//     columns of V's rows 16t + 4g + r and one v_perm per pair of keys makes each operand.
// K's registers are refilled when S is done and V's when O is, so a wave always has about a
// step's bytes in flight.
//
// A sequence's keys are split over workgroups of NW waves when the sequences and key heads
// alone would leave CUs idle; partial results (max, sum, O in 32 bits) are joined by a second
// launch in the order of the splits.
//
// Numerics: fp32 scores, maxima, sums and O.  P is rounded to 16 bits for the product: fp16
// (half a step 2^-11 of the weight) as it is; bf16 (2^-8) as the sum of two bf16 numbers, whose
// second product the idle matrix cores do for nothing.
#include "tk_join.hpp"

namespace tk {
namespace {

struct PagedArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int32_t* table;
  const int32_t* lengths;
  float* part;  // [batch * heads][splits][hd] partial O, then [..][splits][2] max and sum
  float* stats;
  int64_t qs[2], os[2];          // {b, h}
  int64_t ks[3], vs[3];          // {page, head, row}
  int64_t table_stride;
  int batch, heads, kv_heads, group, groups;  // group: heads per key head; groups: blocks of 16 of them
  int hd, pages, page_shift, table_width;
  int window, sinks;  // window 0: all keys
  int splits, per_split;  // tiles of 32 keys
  float scale_log2;
};

// Max / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 that hold one head's keys.
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return pair_max(x);
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return pair_sum(x);
}

template <int DW>
struct Words {
  uint32_t w[DW];
};

template <typename T, int DT, int NW>
__device__ __forceinline__ void paged_body(const PagedArgs& p) {
  typedef typename Elem<T>::x8 x8;
  constexpr int KS = DT / 32;   // 32-wide steps of S^T
  constexpr int CW = DT / 16;   // columns of V per lane
  constexpr int DW = CW / 2;    // the same in words
  constexpr bool SPLIT_P = sizeof(T) == 2 && !__is_same(T, f16);
  __shared__ float o_lds[NW][16][DT];
  __shared__ float m_lds[NW][16], l_lds[NW][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;

  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int grp = id % p.groups;
  id /= p.groups;
  const int kvh = id % p.kv_heads, b = id / p.kv_heads;
  const int h0 = kvh * p.group + grp * 16;          // first query head of the block
  const int nh = min(16, p.group - grp * 16);       // heads of the block

  const int len = min(max(p.lengths[b], 0), p.table_width << p.page_shift);
  const int lo = p.window > 0 ? max(0, len - p.window) : 0;
  // tiles of 32 keys that hold visible ones: those of the sinks, then those of the window
  const int wt = lo >> 5;
  const int st = min((min(p.sinks, lo) + 31) >> 5, wt);
  const int n_tiles = st + ((len + 31) >> 5) - wt;
  const int t_begin = split * p.per_split;
  const int t_end = split == p.splits - 1 ? n_tiles : min(n_tiles, t_begin + p.per_split);

  const int32_t* row = p.table + b * p.table_stride;
  const T* kb = reinterpret_cast<const T*>(p.k) + kvh * p.ks[1];
  const T* vb = reinterpret_cast<const T*>(p.v) + kvh * p.vs[1];

  x8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 32 * s + 8 * g;
    qf[s] = x8{};
    if (c < nh && d < p.hd)
      qf[s] = *reinterpret_cast<const x8*>(reinterpret_cast<const T*>(p.q) + b * p.qs[0] + (h0 + c) * p.qs[1] + d);
  }

  // The page of 16 keys from `key` on, or -1 where the sequence or the cache has none there.
  auto page_of = [&](int key) {
    if (key >= len) return -1;
    const int id = row[key >> p.page_shift];
    return (uint32_t)id < (uint32_t)p.pages ? id : -1;
  };
  auto first_key = [&](int o) { return (o < st ? o : o - st + wt) * 32; };
  const int in_page = (1 << p.page_shift) - 1;

  x8 kf[2][KS];
  Words<DW> vf[8];
  auto load_k = [&](int k0, int p0, int p1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const T* base = kb + (int64_t)max(t ? p1 : p0, 0) * p.ks[0] + (int64_t)(((k0 + 16 * t) & in_page) + c) * p.ks[2];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 32 * s + 8 * g;
        kf[t][s] = x8{};
        if (d < p.hd) kf[t][s] = *reinterpret_cast<const x8*>(base + d);
      }
    }
  };
  auto load_v = [&](int k0, int p0, int p1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const T* base = vb + (int64_t)max(t ? p1 : p0, 0) * p.vs[0];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const T* src = base + (int64_t)(((k0 + 16 * t) & in_page) + 4 * g + r) * p.vs[2];
        Words<DW>& w = vf[4 * t + r];
        if constexpr (DT == 256) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u32x4 x = {0, 0, 0, 0};
            if (128 * e + 8 * c < p.hd) x = *reinterpret_cast<const u32x4*>(src + 128 * e + 8 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) w.w[4 * e + i] = x[i];
          }
        } else {
          const bool in = CW * c < p.hd;
          if constexpr (DW == 4) {
            u32x4 x = {0, 0, 0, 0};
            if (in) x = *reinterpret_cast<const u32x4*>(src + CW * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) w.w[i] = x[i];
          } else if constexpr (DW == 2) {
            u32x2 x = {0, 0};
            if (in) x = *reinterpret_cast<const u32x2*>(src + CW * c);
            w.w[0] = x[0];
            w.w[1] = x[1];
          } else {
            w.w[0] = in ? *reinterpret_cast<const uint32_t*>(src + CW * c) : 0u;
          }
        }
      }
    }
  };

  f32x4 acc[CW];
#pragma unroll
  for (int m = 0; m < CW; ++m) acc[m] = f32x4{};
  float m_run = -INFINITY, l_run = 0.f;
  const float cs = p.scale_log2;

  int o = t_begin + wave;
  int k0 = 0, p0 = -1, p1 = -1;
  if (o < t_end) {
    k0 = first_key(o);
    p0 = page_of(k0);
    p1 = page_of(k0 + 16);
    load_k(k0, p0, p1);
    load_v(k0, p0, p1);
  }
  for (; o < t_end; o += NW) {
    const bool more = o + NW < t_end;
    int k0n = 0, p0n = -1, p1n = -1;
    if (more) {
      k0n = first_key(o + NW);
      p0n = page_of(k0n);
      p1n = page_of(k0n + 16);
    }
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < KS; ++i) s[t] = Elem<T>::mfma16(kf[t][i], qf[i], i == 0 ? f32x4{} : s[t]);
    if (more) load_k(k0n, p0n, p1n);

    // keys that the token does not see, on the tiles that have any
    const bool edge = k0 + 32 > len || (k0 < lo && k0 + 32 > p.sinks) || p0 < 0 || p1 < 0;
    uint32_t ok = 0xff;
    if (edge) {
      ok = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = k0 + 16 * t + 4 * g + r;
          const bool see = key < len && (key >= lo || key < p.sinks) && (t ? p1 : p0) >= 0;
          ok |= (uint32_t)see << (4 * t + r);
          if (!see) s[t][r] = -INFINITY;
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    const float m_new = fmaxf(m_run, quad_max(mx) * cs);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    m_run = m_new;
    float e[8];
    l_run *= alpha;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], cs, -m_use));
      l_run += e[i];
    }
    x8 pf, pl;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pf[i] = (T)e[i];
      if (SPLIT_P) pl[i] = (T)(e[i] - (float)pf[i]);
    }
#pragma unroll
    for (int m = 0; m < CW; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[m][r] *= alpha;
    if (edge) {  // whatever lies in rows that are not seen times a weight of 0 must be 0
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < DW; ++w) vf[i].w[w] = (ok >> i) & 1 ? vf[i].w[w] : 0u;
    }
#pragma unroll
    for (int m = 0; m < CW; ++m) {
      u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        a[i] = __builtin_amdgcn_perm(vf[2 * i + 1].w[m >> 1], vf[2 * i].w[m >> 1], m & 1 ? 0x07060302u : 0x05040100u);
      const x8 va = __builtin_bit_cast(x8, a);
      acc[m] = Elem<T>::mfma16(va, pf, acc[m]);
      if (SPLIT_P) acc[m] = Elem<T>::mfma16(va, pl, acc[m]);
    }
    if (more) load_v(k0n, p0n, p1n);
    k0 = k0n;
    p0 = p0n;
    p1 = p1n;
  }

  // ---- the waves' results, rescaled to the common maximum and added in wave order ----
  l_run = quad_sum(l_run);
#pragma unroll
  for (int m = 0; m < CW; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = 4 * g + r;
      o_lds[wave][c][DT == 256 ? 128 * (m >> 3) + 8 * n + (m & 7) : CW * n + m] = acc[m][r];
    }
  if (g == 0) {
    m_lds[wave][c] = m_run;
    l_lds[wave][c] = l_run;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * DT; i += NW * 64) {
    const int h = i / DT, d = i % DT;
    if (d >= p.hd) continue;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) m_all = fmaxf(m_all, m_lds[w][h]);
    const float m_ref = m_all == -INFINITY ? 0.f : m_all;
    float sum = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_lds[w][h] - m_ref);
      sum += f * o_lds[w][h][d];
      l += f * l_lds[w][h];
    }
    if (p.splits == 1) {
      T* out = reinterpret_cast<T*>(p.o) + b * p.os[0] + (h0 + h) * p.os[1] + d;
      *out = (T)(l == 0.f ? 0.f : sum / l);
    } else {
      const int64_t part = ((int64_t)b * p.heads + h0 + h) * p.splits + split;
      if (m_all != -INFINITY) p.part[part * p.hd + d] = sum;
      if (d == 0) {
        p.stats[2 * part] = m_all;
        p.stats[2 * part + 1] = l;
      }
    }
  }
}

template <typename T, int DT, int NW>
__global__ __launch_bounds__(NW * 64) void paged_attn_kernel(PagedArgs p) {
  paged_body<T, DT, NW>(p);
}

constexpr int kPagedWaves = 4;

// Tiles of 32 keys a workgroup takes, and the splits that this makes of a sequence of max_length keys.
struct PagedPlan {
  int64_t splits, per_split;
};
PagedPlan paged_plan(int64_t blocks, int64_t max_length, int64_t window, int64_t sinks, bool batch_invariant) {
  int64_t keys = max_length;
  if (window > 0 && keys > window + sinks) keys = window + sinks;
  const int64_t tiles = (keys + 31) / 32 + (window > 0 ? 2 : 0);  // a window may begin and end inside tiles
  int64_t per = 32;
  if (!batch_invariant) {
    const int64_t want = (1024 + blocks - 1) / blocks;  // splits that give each CU four workgroups
    per = (tiles + want - 1) / want;
    per = (per + kPagedWaves - 1) / kPagedWaves * kPagedWaves;
    if (per < 2 * kPagedWaves) per = 2 * kPagedWaves;
  }
  int64_t splits = (tiles + per - 1) / per;
  if (splits < 1) splits = 1;
  return {splits, per};
}

template <typename T>
int launch_paged(const PagedArgs& p, int64_t grid, hipStream_t st) {
  constexpr int NW = kPagedWaves;
  const dim3 g((unsigned)grid), blk(NW * 64);
  if (p.hd <= 32) hipLaunchKernelGGL((paged_attn_kernel<T, 32, NW>), g, blk, 0, st, p);
  else if (p.hd <= 64) hipLaunchKernelGGL((paged_attn_kernel<T, 64, NW>), g, blk, 0, st, p);
  else if (p.hd <= 128) hipLaunchKernelGGL((paged_attn_kernel<T, 128, NW>), g, blk, 0, st, p);
  else hipLaunchKernelGGL((paged_attn_kernel<T, 256, NW>), g, blk, 0, st, p);
  int rc = check_launch("tk_paged_attn");
  if (rc != TK_OK || p.splits == 1) return rc;
  JoinArgs j{};
  j.part = p.part;
  j.stats = p.stats;
  j.o = p.o;
  j.os[0] = p.os[0];
  j.os[1] = p.os[1];
  j.heads = p.heads;
  j.q_len = 1;
  j.hd = p.hd;
  j.splits = p.splits;
  return launch_join<T>("tk_paged_attn", j, (int64_t)p.batch * p.heads, st);
}

}  // namespace
}  // namespace tk

using namespace tk;

namespace {

int check_paged_shape(const char* fn, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                      int64_t max_length, int64_t window, int64_t sinks) {
  TK_REQUIRE(batch >= 0 && heads >= 0 && kv_heads >= 0 && head_dim >= 0 && max_length >= 0 && window >= 0 && sinks >= 0,
             TK_ERR_ARG, "%s: negative size", fn);
  TK_REQUIRE(batch < (1ll << 31) && heads < (1ll << 31) && kv_heads < (1ll << 31) && max_length < (1ll << 30) &&
                 window < (1ll << 30) && sinks < (1ll << 30),
             TK_ERR_ARG, "%s: size out of range", fn);
  TK_REQUIRE(kv_heads == 0 ? heads == 0 : heads % kv_heads == 0, TK_ERR_ARG,
             "%s: heads=%lld is no multiple of kv_heads=%lld", fn, (long long)heads, (long long)kv_heads);
  TK_REQUIRE(head_dim <= 256 && head_dim % 8 == 0, TK_ERR_UNSUPPORTED,
             "%s: head_dim=%lld is no multiple of 8 up to 256", fn, (long long)head_dim);
  TK_REQUIRE(batch == 0 || heads == 0 || batch * heads < (1ll << 24), TK_ERR_UNSUPPORTED,
             "%s: batch * heads = %lld rows above 2^24", fn, (long long)(batch * heads));
  return TK_OK;
}

int64_t paged_blocks(int64_t batch, int64_t heads, int64_t kv_heads) {
  return kv_heads == 0 ? 0 : batch * kv_heads * ((heads / kv_heads + 15) / 16);
}

}  // namespace

extern "C" int64_t tk_paged_attn_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           int64_t max_length, int64_t window, int64_t sinks, int batch_invariant) {
  const int rc = check_paged_shape("tk_paged_attn_workspace", batch, heads, kv_heads, head_dim, max_length, window,
                                   sinks);
  if (rc != TK_OK) return rc;
  const int64_t blocks = paged_blocks(batch, heads, kv_heads);
  if (blocks == 0) return 0;
  const PagedPlan plan = paged_plan(blocks, max_length, window, sinks, batch_invariant != 0);
  return plan.splits == 1 ? 0 : batch * heads * plan.splits * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int tk_paged_attn(const void* q, const int64_t* q_strides, const void* k_pages, const int64_t* k_strides,
                             const void* v_pages, const int64_t* v_strides, void* out, const int64_t* o_strides,
                             int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                             int64_t pages, int64_t page_size, const int32_t* table, int64_t table_stride,
                             int64_t table_width, const int32_t* lengths, int64_t max_length, float scale,
                             int64_t window, int64_t sinks, int batch_invariant, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const int rc = check_paged_shape("tk_paged_attn", batch, heads, kv_heads, head_dim, max_length, window, sinks);
  if (rc != TK_OK) return rc;
  TK_REQUIRE(dtype == TK_F16 || dtype == TK_BF16, TK_ERR_ARG, "tk_paged_attn: dtype %d is not TK_F16 or TK_BF16", dtype);
  TK_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, TK_ERR_UNSUPPORTED,
             "tk_paged_attn: page_size=%lld is no power of two from 16 to 1024", (long long)page_size);
  TK_REQUIRE(pages >= 0 && pages < (1ll << 31) && table_width >= 0 && table_width * page_size < (1ll << 30),
             TK_ERR_ARG, "tk_paged_attn: pages or table width out of range");
  TK_REQUIRE(batch <= 1 || table_stride >= table_width, TK_ERR_ARG, "tk_paged_attn: table_stride < table_width");
  TK_REQUIRE(scale > 0.f && scale <= 3.0e38f, TK_ERR_ARG, "tk_paged_attn: scale must be positive and finite");
  if (batch == 0 || heads == 0 || head_dim == 0) return TK_OK;
  TK_REQUIRE(q && out && lengths && q_strides && k_strides && v_strides && o_strides &&
                 ((k_pages && v_pages) || pages == 0) && (table || table_width == 0),
             TK_ERR_ARG, "tk_paged_attn: null pointer");
  auto al = [](const void* ptr, uintptr_t a) { return ((uintptr_t)ptr % a) == 0; };
  TK_REQUIRE(al(q, 16) && al(k_pages, 16) && al(v_pages, 16) && al(out, 2) && q_strides[0] % 8 == 0 &&
                 q_strides[1] % 8 == 0,
             TK_ERR_UNSUPPORTED, "tk_paged_attn: rows of q, k_pages and v_pages must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    TK_REQUIRE(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, TK_ERR_UNSUPPORTED,
               "tk_paged_attn: rows of q, k_pages and v_pages must be 16-byte aligned");
  const int64_t blocks = paged_blocks(batch, heads, kv_heads);
  // the last split takes what is past max_length: with one order for every call there must be nothing
  if (batch_invariant && max_length < table_width * page_size) max_length = table_width * page_size;
  const PagedPlan plan = paged_plan(blocks, max_length, window, sinks, batch_invariant != 0);
  TK_REQUIRE(blocks * plan.splits < (1ll << 31), TK_ERR_UNSUPPORTED, "tk_paged_attn: too many workgroups");
  const int64_t rows = batch * heads;
  if (plan.splits > 1) {
    const int64_t need = rows * plan.splits * (head_dim + 2) * (int64_t)sizeof(float);
    TK_REQUIRE(workspace && al(workspace, 16) && workspace_bytes >= need, TK_ERR_ARG,
               "tk_paged_attn: workspace of %lld bytes, 16-byte aligned, needed", (long long)need);
  }
  PagedArgs p{};
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.o = out;
  p.table = table;
  p.lengths = lengths;
  p.part = reinterpret_cast<float*>(workspace);
  p.stats = p.part ? p.part + rows * plan.splits * head_dim : nullptr;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = o_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  p.table_stride = table_stride;
  p.batch = (int)batch;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads);
  p.groups = (p.group + 15) / 16;
  p.hd = (int)head_dim;
  p.pages = (int)pages;
  p.page_shift = __builtin_ctzll((unsigned long long)page_size);
  p.table_width = pages > 0 ? (int)table_width : 0;
  p.window = (int)window;
  p.sinks = (int)sinks;
  p.splits = (int)plan.splits;
  p.per_split = (int)plan.per_split;
  p.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t st = as_stream(stream);
  return dtype == TK_F16 ? launch_paged<f16>(p, blocks * plan.splits, st)
                         : launch_paged<bf16>(p, blocks * plan.splits, st);
}
