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
// step's bytes in flight.  Measured: 64 sequences of 16384 tokens, 4 key heads of 128, 6.1 TB/s; 200 of
// about 1000 visible ones, 16 heads of 64, 5.5; 64 of 100 to 4096, 4 heads of 128 bf16, 4.6 (61 us); one
// of 100000, 2 heads of 128, 5.1 (20 us) and 4 us for the join.  Fixed cost of a launch: 4.2 us.
//
// Where the sequences and key heads alone would leave CUs idle, every sequence's keys are split
// over workgroups (paged_share), and a second launch joins their results (tk_join.hpp).
//
// Numerics: fp32 scores, references, sums and O.  P goes into the product as the sum of two 16-bit numbers, the
// second the first one's rounding error, whose product the idle matrix cores do (fp16: +1.2 % of the time over 20
// shapes, 4.18 -> 4.28 us for a single short sequence, nothing where HBM bounds).  What is left is 2^-16 of a weight in bf16; in fp16, where the largest is 2^15 (weight_ref), 2^-22 of weights down to 2^-18 of
// the wave's largest, and at most 2^-40 of that one below.
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
  float* part;   // partial results (tk_join.hpp)
  float* stats;
  int32_t* plan;
  int64_t qs[2], os[2];          // {b, h}
  int64_t ks[3], vs[3];          // {page, head, row}
  int64_t table_stride;
  int batch, heads, kv_heads, group, groups;  // group: heads per key head; groups: blocks of 16 of them
  int hd, pages, page_shift, table_width;
  int window, sinks;  // window 0: all keys
  int workers;  // workgroups per key head and block of heads
  bool shared;  // paged_share; else one worker per sequence, or fixed ones
  bool fill;    // paged_share: as many shares as there are workers
  int least;    // tiles of the smallest share
  int fixed;    // > 0: shares of this many tiles, workers / batch of them per sequence
  float scales[3];  // weight_ref
};

// The tiles of 32 keys that hold visible ones: those of the sinks, then those of the window.
struct PagedTiles {
  int len, lo, wt, st, n;
  __device__ __forceinline__ PagedTiles(const PagedArgs& p, int length) {
    len = min(max(length, 0), p.table_width << p.page_shift);
    lo = p.window > 0 ? max(0, len - p.window) : 0;
    wt = lo >> 5;
    st = min((min(p.sinks, lo) + 31) >> 5, wt);
    n = st + ((len + 31) >> 5) - wt;
  }
  __device__ __forceinline__ int key(int t) const { return (t < st ? t : t - st + wt) * 32; }
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

template <bool B>
struct BoolOf {
  static constexpr bool value = B;
};

// Sum over the wave's lanes, in every lane, without LDS: quads and rows of 16 by DPP, then the rows.
__device__ __forceinline__ int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, true);   // lane ^ 1
  x += __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, true);   // lane ^ 2
  x += __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);  // 7 - lane of each 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true);  // 15 - lane of each 16
  return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) +
         __builtin_amdgcn_readlane(x, 48);
}

// What a worker takes: share `index` of `count` of sequence b (of `len` tokens); `first`: the worker of share 0.
struct PagedShare {
  int b, len, index, count, first;
};

// Sequences of different lengths are cut into shares of nearly one size, so that every CU has the same to
// do: sequence b of n_b tiles into ceil(n_b / size) equal ones.  With fewer sequences than CUs (p.fill) size
// is the smallest (in steps of the workgroup's waves) at which there are no more shares than workers: with
// one workgroup per CU in all, any share too many shares its CU (12 sequences of 36254 tokens, 4 key heads
// of 128, in 240 workgroups take 153 us, in 288 206).  With more, only sequences of more than twice what
// a CU has on average are cut, which otherwise end long after all the others.  Every wave finds its
// worker's place from all lengths, at most kShareRows of them, a few registers.
constexpr int kShareRows = 1024;
template <int NW>
__device__ __forceinline__ PagedShare paged_share(const PagedArgs& p, int worker) {
  constexpr int kPer = kShareRows / 64;
  const int lane = threadIdx.x & 63;
  int len[kPer], tiles[kPer];
  int total = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (64 * i >= p.batch) continue;
    const int b = 64 * i + lane;
    len[i] = b < p.batch ? p.lengths[b] : 0;
    tiles[i] = b < p.batch ? max(PagedTiles(p, len[i]).n, 1) : 0;
    total += tiles[i];
  }
  total = wave_sum(total);
  // ceil(n_b / size) add up to less than total / size + batch
  int low = max(total / (p.workers * NW), p.least / NW), high = max(total / ((p.workers - p.batch) * NW) + 1, low);
  while (p.fill && low < high) {
    const int mid = (low + high) / 2;
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (64 * i < p.batch) n += ((uint32_t)tiles[i] + mid * NW - 1) / (uint32_t)(mid * NW);
    if (wave_sum(n) <= p.workers) high = mid;
    else low = mid + 1;
  }
  const uint32_t size = high * NW;
  PagedShare r = {-1, 0, 0, 1, 0};
  int before = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (64 * i >= p.batch) continue;
    const int n = ((uint32_t)tiles[i] + size - 1) / size;
    int incl = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(incl, off);
      if (lane >= off) incl += y;
    }
    const int first = before + incl - n;
    const uint64_t mine = __ballot(worker >= first && worker < first + n);
    if (mine) {
      const int src = __builtin_ctzll(mine);
      r.b = 64 * i + src;
      r.len = __builtin_amdgcn_readlane(len[i], src);
      r.first = __builtin_amdgcn_readlane(first, src);
      r.count = __builtin_amdgcn_readlane(n, src);
      r.index = worker - r.first;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return r;
}

// The waves' results: rows of 4 floats more, so that 16 heads' 16-byte pieces fall on different banks.
template <int DT, int NW>
struct PagedLds {
  float o[NW][16][DT + 4];
  float m[NW][16], l[NW][16];
};

// Tiles [t_begin, t_end) of sequence b for query heads h0 .. h0 + nh of key head kvh: the rows' output if
// that is all of the sequence, else a partial result in the worker's slots.
template <typename T, int DT, int NW>
__device__ __forceinline__ void paged_segment(const PagedArgs& p, PagedLds<DT, NW>& lds, int kvh, int h0, int nh, int b,
                                              const PagedTiles& tiles, int t_begin, int t_end, bool whole, int worker) {
  typedef typename Elem<T>::x8 x8;
  constexpr int KS = DT / 32;   // 32-wide steps of S^T
  constexpr int CW = DT / 16;   // columns of V per lane
  constexpr int DW = CW / 2;    // the same in words

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int len = tiles.len, lo = tiles.lo;

  // A step's addresses are a scalar (page and row of 16 keys) plus a lane's 32-bit offset.  Columns past
  // head_dim re-read the last ones: they meet zeros of Q or are not stored.
  const char* kb = reinterpret_cast<const char*>(p.k) + 2 * kvh * p.ks[1];
  const char* vb = reinterpret_cast<const char*>(p.v) + 2 * kvh * p.vs[1];
  const int64_t k_page = 2 * p.ks[0], k_row = 2 * p.ks[2], v_page = 2 * p.vs[0], v_row = 2 * p.vs[2];
  const int in_page = (1 << p.page_shift) - 1;
  constexpr int VL = DT == 256 ? 2 : 1;  // loads of a row of V
  uint32_t k_off[KS], v_off[4][VL];
#pragma unroll
  for (int s = 0; s < KS; ++s) k_off[s] = (uint32_t)(c * k_row) + 2 * min(32 * s + 8 * g, p.hd - 8);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      const int col = DT == 256 ? 128 * e + 8 * c : CW * c;
      v_off[r][e] = (uint32_t)((4 * g + r) * v_row) + 2 * min(col, p.hd - CW / VL);
    }

  x8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 32 * s + 8 * g;
    qf[s] = x8{};
    if (c < nh && d < p.hd)
      qf[s] = *reinterpret_cast<const x8*>(reinterpret_cast<const T*>(p.q) + b * p.qs[0] + (h0 + c) * p.qs[1] + d);
  }

  // Lane l holds the page of the 16 keys l & 1 of the wave's step l >> 1 of 32, or -1 where the cache has
  // none: one load for 32 steps, made 32 steps ahead.  (A load of a step's pages in that step waits for
  // every load before it.)  Without a window it does not wait for the sequence's length.
  const int steps = t_begin + wave < t_end ? (t_end - t_begin - wave + NW - 1) / NW : 0;
  const int32_t* row = p.table + b * p.table_stride;
  auto load_pages = [&](int step) {
    const int key = tiles.key(t_begin + wave + (step + (lane >> 1)) * NW) + 16 * (lane & 1);
    const int id = (key >> p.page_shift) < p.table_width ? row[key >> p.page_shift] : -1;
    return (uint32_t)id < (uint32_t)p.pages ? id : -1;
  };
  auto page = [&](int pg, int step, int half, int key) {
    const int id = __builtin_amdgcn_readlane(pg, 2 * (step & 31) + half);
    return key + 16 * half < len ? id : -1;
  };

  x8 kf[2][KS];
  uint32_t vf[8][DW];
  auto load_k = [&](int k0, int p0, int p1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* base = kb + max(t ? p1 : p0, 0) * k_page + ((k0 + 16 * t) & in_page) * k_row;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[t][s] = *reinterpret_cast<const x8*>(base + k_off[s]);
    }
  };
  auto load_v = [&](int k0, int p0, int p1) {
    typedef uint32_t words __attribute__((ext_vector_type(DW / VL)));
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* base = vb + max(t ? p1 : p0, 0) * v_page + ((k0 + 16 * t) & in_page) * v_row;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const words x = *reinterpret_cast<const words*>(base + v_off[r][e]);
          __builtin_memcpy(&vf[4 * t + r][e * (DW / VL)], &x, sizeof(x));
        }
    }
  };

  f32x4 acc[CW];
#pragma unroll
  for (int m = 0; m < CW; ++m) acc[m] = f32x4{};
  float m_run = -INFINITY, l_run = 0.f;
  const float cs = p.scales[0];

  // One step: the keys from k0 on are in kf and vf; those from `k0n` on follow, if there are more.
  auto step = [&](auto more, int k0, int p0, int p1, int k0n, int p0n, int p1n) {
    f32x4 s[2];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = Elem<T>::mfma16(kf[t][i], qf[i], i == 0 ? f32x4{} : s[t]);
    // (the barriers keep the loads from being hoisted into registers of their own: 228 + 64 of them at DT = 128)
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (decltype(more)::value) load_k(k0n, p0n, p1n);
    __builtin_amdgcn_sched_barrier(0);

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
    const float m_new = fmaxf(m_run, weight_ref<T, 15>(quad_max(mx), p.scales));
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
      pl[i] = (T)(e[i] - (float)pf[i]);
    }
#pragma unroll
    for (int m = 0; m < CW; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[m][r] *= alpha;
    if (edge) {  // whatever lies in rows that are not seen times a weight of 0 must be 0
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < DW; ++w) vf[i][w] = (ok >> i) & 1 ? vf[i][w] : 0u;
    }
#pragma unroll
    for (int m = 0; m < CW; ++m) {
      u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        a[i] = __builtin_amdgcn_perm(vf[2 * i + 1][m >> 1], vf[2 * i][m >> 1], m & 1 ? 0x07060302u : 0x05040100u);
      const x8 va = __builtin_bit_cast(x8, a);
      acc[m] = Elem<T>::mfma16(va, pf, acc[m]);
      acc[m] = Elem<T>::mfma16(va, pl, acc[m]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (decltype(more)::value) load_v(k0n, p0n, p1n);
    __builtin_amdgcn_sched_barrier(0);
  };

  if (steps > 0) {
    int pg = load_pages(0), pg_next = -1;
    if (steps > 32) pg_next = load_pages(32);
    int k0 = tiles.key(t_begin + wave);
    int p0 = page(pg, 0, 0, k0), p1 = page(pg, 0, 1, k0);
    load_k(k0, p0, p1);
    load_v(k0, p0, p1);
    for (int i = 1; i < steps; ++i) {
      if ((i & 31) == 0) {
        pg = pg_next;
        if (i + 32 < steps) pg_next = load_pages(i + 32);
      }
      const int k0n = tiles.key(t_begin + wave + i * NW);
      const int p0n = page(pg, i, 0, k0n), p1n = page(pg, i, 1, k0n);
      step(BoolOf<true>(), k0, p0, p1, k0n, p0n, p1n);
      k0 = k0n;
      p0 = p0n;
      p1 = p1n;
    }
    step(BoolOf<false>(), k0, p0, p1, 0, -1, -1);
  }

  // ---- the waves' results, rescaled to the largest reference and added in wave order ----
  l_run = quad_sum(l_run);
  constexpr int VW = CW < 4 ? CW : 4;  // neighbouring columns written at once
  typedef float vec __attribute__((ext_vector_type(VW)));
  if (c < nh) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int m = 0; m < CW; m += VW) {
        const int n = 4 * g + r;
        vec x;
#pragma unroll
        for (int i = 0; i < VW; ++i) x[i] = acc[m + i][r];
        *reinterpret_cast<vec*>(&lds.o[wave][c][DT == 256 ? 128 * (m >> 3) + 8 * n + (m & 7) : CW * n + m]) = x;
      }
    if (g == 0) {
      lds.m[wave][c] = m_run;
      lds.l[wave][c] = l_run;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * (DT / 4); i += NW * 64) {
    const int h = i / (DT / 4), d = i % (DT / 4) * 4;
    if (d >= p.hd) continue;
    float f[NW], m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = lds.m[w][h];
      m_all = fmaxf(m_all, f[w]);
    }
    const float m_ref = m_all == -INFINITY ? 0.f : m_all;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = __builtin_amdgcn_exp2f(f[w] - m_ref);
      const f32x4 o = *reinterpret_cast<const f32x4*>(&lds.o[w][h][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(f[w], o[e], sum[e]);
      l = fmaf(f[w], lds.l[w][h], l);
    }
    if (whole) {
      T* out = reinterpret_cast<T*>(p.o) + b * p.os[0] + (h0 + h) * p.os[1] + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = (T)(l == 0.f ? 0.f : sum[e] / l);
    } else {
      const int64_t part = (int64_t)worker * p.heads + h0 + h;
      if (m_all != -INFINITY) *reinterpret_cast<f32x4*>(p.part + part * p.hd + d) = sum;
      if (d == 0) {
        p.stats[2 * part] = m_all;
        p.stats[2 * part + 1] = l;
      }
    }
  }
}

// SHARED: paged_share; else one worker per sequence, or a fixed number of them (batch_invariant).
template <typename T, int DT, int NW, bool SHARED>
__device__ __forceinline__ void paged_body(const PagedArgs& p) {
  __shared__ PagedLds<DT, NW> lds;
  const int hg = blockIdx.x % (p.kv_heads * p.groups), worker = blockIdx.x / (p.kv_heads * p.groups);
  const int kvh = hg / p.groups, grp = hg % p.groups;
  const int h0 = kvh * p.group + grp * 16, nh = min(16, p.group - grp * 16);
  PagedShare share;
  int per;
  if constexpr (SHARED) {
    share = paged_share<NW>(p, worker);
    if (share.b < 0) return;
  } else {
    const int count = p.workers / p.batch, b = worker / count;
    share = {b, p.lengths[b], worker % count, count, b * count};
  }
  const PagedTiles tiles(p, share.len);
  if constexpr (SHARED) per = (tiles.n + share.count * NW - 1) / (share.count * NW) * NW;  // whole steps of the waves
  else per = p.fixed;
  if (share.count > 1 && hg == 0 && share.index == 0 && threadIdx.x == 0) p.plan[2 * share.b] = worker;
  if (p.plan && hg == 0 && share.index == 0 && threadIdx.x == 0) p.plan[2 * share.b + 1] = share.count;
  const int t_begin = share.index * per, t_end = share.index == share.count - 1 ? tiles.n : min(tiles.n, t_begin + per);
  paged_segment<T, DT, NW>(p, lds, kvh, h0, nh, share.b, tiles, t_begin, t_end, share.count == 1, worker);
}

template <typename T, int DT, int NW, bool SHARED>
__global__ __launch_bounds__(NW * 64, DT <= 128 ? 2 : 1) void paged_attn_kernel(PagedArgs p) {
  paged_body<T, DT, NW, SHARED>(p);
}

constexpr int kPagedWaves = 4;

// Workers per key head and block of 16 heads; the others: PagedArgs.
struct PagedPlan {
  int64_t workers, fixed;
  bool shared, fill;
};
constexpr int64_t kPagedBlocks = 256;             // one workgroup per CU
constexpr int64_t kPagedLong = 256;               // tiles from which on one sequence may outlast all others
constexpr int64_t kPagedLeast = 2 * kPagedWaves;  // tiles of the smallest share: two steps of every wave
PagedPlan paged_plan(int64_t batch, int64_t per_seq, int64_t max_length, int64_t window, int64_t sinks,
                     bool batch_invariant) {
  int64_t keys = max_length;
  if (window > 0 && keys > window + sinks) keys = window + sinks;
  const int64_t tiles = (keys + 31) / 32 + (window > 0 ? 2 : 0);  // a window may begin and end inside tiles
  if (batch_invariant) {
    const int64_t per = 32, n = (tiles + per - 1) / per;
    return {batch * (n > 1 ? n : 1), per, false, false};
  }
  const int64_t most = (tiles + kPagedLeast - 1) / kPagedLeast;  // shares of the longest sequence
  // From half the CUs on, a split of every sequence gains less than the launch that joins it takes: 186
  // sequences of 676 to 917 tokens, one key head of 64, in whole ones 10.7 us, split 16.8; 17 sequences of
  // 4000, 8 key heads of 128 57 and 70.  (Below: 2 sequences of 2000 tokens, 2 key heads of 128, 10 us split,
  // 17 whole.)  Only where a sequence may be long enough to outlast all others are such ones cut: 199
  // of 100 tokens and one of 60000, one key head of 128, take 25.6 us, whole 524.
  const int64_t whole = kPagedBlocks / 2 / per_seq;  // sequences
  if (batch >= whole) {
    if (tiles < kPagedLong || batch > kShareRows) return {batch, 0, false, false};
    return {batch + (whole > 1 ? whole : 1), 0, true, false};
  }
  if (most <= 1) return {batch, 0, false, false};
  const int64_t full = kPagedBlocks / per_seq, workers = full < batch * (most + 1) ? full : batch * (most + 1);
  return {workers, 0, true, true};
}

template <typename T, int DT>
void launch_paged_dim(const PagedArgs& p, int64_t grid, hipStream_t st) {
  const dim3 g((unsigned)grid), blk(kPagedWaves * 64);
  if (p.shared) hipLaunchKernelGGL((paged_attn_kernel<T, DT, kPagedWaves, true>), g, blk, 0, st, p);
  else hipLaunchKernelGGL((paged_attn_kernel<T, DT, kPagedWaves, false>), g, blk, 0, st, p);
}

template <typename T>
int launch_paged(const PagedArgs& p, int64_t grid, hipStream_t st) {
  if (p.hd <= 32) launch_paged_dim<T, 32>(p, grid, st);
  else if (p.hd <= 64) launch_paged_dim<T, 64>(p, grid, st);
  else if (p.hd <= 128) launch_paged_dim<T, 128>(p, grid, st);
  else launch_paged_dim<T, 256>(p, grid, st);
  const int rc = check_launch("tk_paged_attn");
  if (rc != TK_OK || !p.plan) return rc;
  JoinArgs j{};
  j.part = p.part;
  j.stats = p.stats;
  j.o = p.o;
  j.os[0] = p.os[0];
  j.os[1] = p.os[1];
  j.heads = p.heads;
  j.q_len = 1;
  j.hd = p.hd;
  j.plan = p.plan;
  j.splits = p.workers / p.batch;
  j.rows = (int64_t)p.batch * p.heads;
  return launch_join<T>("tk_paged_attn", j, p.fixed > 0, st);
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

// Workgroups that a sequence takes at least: one per key head and 16 query heads that share it.
int64_t per_sequence(int64_t heads, int64_t kv_heads) { return kv_heads * ((heads / kv_heads + 15) / 16); }

// A partial result per worker and head, then every sequence's {first worker, workers}.
int64_t paged_workspace(const PagedPlan& plan, int64_t batch, int64_t heads, int64_t head_dim) {
  if (plan.workers == batch) return 0;  // one per sequence writes the output
  return plan.workers * heads * (head_dim + 2) * (int64_t)sizeof(float) + 2 * batch * (int64_t)sizeof(int32_t);
}

}  // namespace

extern "C" int64_t tk_paged_attn_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           int64_t max_length, int64_t window, int64_t sinks, int batch_invariant) {
  const int rc = check_paged_shape("tk_paged_attn_workspace", batch, heads, kv_heads, head_dim, max_length, window,
                                   sinks);
  if (rc != TK_OK) return rc;
  if (batch == 0 || heads == 0) return 0;
  return paged_workspace(paged_plan(batch, per_sequence(heads, kv_heads), max_length, window, sinks,
                                    batch_invariant != 0),
                         batch, heads, head_dim);
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
  TK_REQUIRE(batch == 0 || table_width * page_size <= (1ll << 34) / batch, TK_ERR_UNSUPPORTED,
             "tk_paged_attn: a table of more than 2^34 tokens");
  TK_REQUIRE(batch <= 1 || table_stride >= table_width, TK_ERR_ARG, "tk_paged_attn: table_stride < table_width");
  TK_REQUIRE(scale > 0.f && scale <= kMaxScale, TK_ERR_ARG,
             "tk_paged_attn: scale must be positive and at most 2.3e38");
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
  TK_REQUIRE(k_strides[2] >= 0 && k_strides[2] < (1ll << 26) && v_strides[2] >= 0 && v_strides[2] < (1ll << 26),
             TK_ERR_UNSUPPORTED, "tk_paged_attn: rows of a page 2^26 elements apart or more");
  // the last share takes what is past max_length: with one order for every call there must be nothing
  if (batch_invariant && max_length < table_width * page_size) max_length = table_width * page_size;
  const int64_t per_seq = per_sequence(heads, kv_heads);
  const PagedPlan plan = paged_plan(batch, per_seq, max_length, window, sinks, batch_invariant != 0);
  const int64_t need = paged_workspace(plan, batch, heads, head_dim);
  TK_REQUIRE(per_seq * plan.workers <= kMaxGroups &&
                 (need == 0 || join_grid(batch * heads, head_dim, plan.workers / batch, plan.fixed > 0) <= kMaxGroups),
             TK_ERR_UNSUPPORTED, "tk_paged_attn: too many workgroups");
  TK_REQUIRE(need == 0 || (workspace && al(workspace, 16) && workspace_bytes >= need), TK_ERR_ARG,
             "tk_paged_attn: workspace of %lld bytes, 16-byte aligned, needed", (long long)need);
  PagedArgs p{};
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.o = out;
  p.table = table;
  p.lengths = lengths;
  if (need > 0) {
    p.part = reinterpret_cast<float*>(workspace);
    p.stats = p.part + plan.workers * heads * head_dim;
    p.plan = reinterpret_cast<int32_t*>(p.stats + 2 * plan.workers * heads);
  }
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
  p.workers = (int)plan.workers;
  p.shared = plan.shared;
  p.fill = plan.fill;
  p.least = (int)kPagedLeast;
  p.fixed = (int)plan.fixed;
  set_scales(p.scales, scale);
  hipStream_t st = as_stream(stream);
  return dtype == TK_F16 ? launch_paged<f16>(p, per_seq * plan.workers, st)
                         : launch_paged<bf16>(p, per_seq * plan.workers, st);
}
