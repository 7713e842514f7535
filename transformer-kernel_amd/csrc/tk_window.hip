// Causal attention over a sliding window of keys and a few first ones (sinks) that stay visible.
//
// The query row i of q_len sits at position p = k_len - q_len + i and sees key j when
//   j <= p  and  (j > p - window  or  j < sinks)  and  key_valid[b, j];
// a row that sees nothing is 0.  heads / kv_heads query heads share a key head.
//
// Bound by the matrix cores (4 head_dim flops per visible pair) and the exponentials beside
// them; only the 64-key tiles that some row of a workgroup sees are visited: those of the
// sinks, then those of the window.  A workgroup has 32 rows of one head per wave; K and V tiles
// go global -> LDS by direct copies one tile ahead, two slots each, one barrier per tile.
//
// As in tk_attention.hip a wave computes S^T = K . Q^T (a lane holds one query row's scores, the
// running maximum is one lane-pair exchange) and O^T = V^T . P^T with the accumulator's keys as
// the product's k slots and V^T from transposed LDS reads.  The weights' reference (weight_ref) is
// raised only when a tile's largest score passes that of the tile that set it by more than 2^8, harmless
// in fp32 and in 16-bit P, and the rescale of O is skipped on most tiles.
//
// Numerics: fp32 scores, references, sums, O; P rounded to the inputs' type for the product, the sum taken
// of the rounded weights, so that they add up to 1.  Half a step is 2^-8 of the weight in bf16; in fp16,
// with weights up to 2^15, 2^-11 of those down to 2^-21 of the largest when the reference was set, and 2^-32
// of that one below.
#include "tk_attn_tile.hpp"
#include "tk_join.hpp"

namespace tk {
namespace {

struct WindowArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const uint8_t* kv;  // nullable [batch][k_len]
  int64_t kvs;
  int64_t qs[3], ks[3], vs[3], os[3];  // elements, {b, h, s}
  int batch, heads, group, q_len, k_len, hd, window, sinks;
  int n_qt;
  int unit;               // window_split_kernel: heads whose rows, one head's after another's, make one list
  int splits, per_split;  //   and key tiles of a workgroup
  float* part;            // its results where splits > 1 (tk_join.hpp)
  float* stats;
  float scales[3];        // weight_ref
};

// The key tiles that rows at positions [first, last] see: those of the sinks, then those of the windows.
template <int BN>
struct TileList {
  int st, wt, n;
  __device__ __forceinline__ TileList(const WindowArgs& p, int first, int last) {
    const int lo = max(0, first - p.window + 1);
    wt = lo / BN;
    st = min((min(p.sinks, lo) + BN - 1) / BN, wt);
    n = st + last / BN + 1 - wt;
  }
  __device__ __forceinline__ int key(int t) const { return (t < st ? t : t - st + wt) * BN; }
};

template <typename T, int DT, int BN, int NW, bool KMASK>
__device__ __forceinline__ void window_body(const WindowArgs& p) {
  typedef typename Elem<T>::x8 x8;
  typedef typename Elem<T>::x4 x4;
  constexpr int NB = BN / 32;
  constexpr int RB = DT * 2;
  constexpr int CPR = RB / 16;
  constexpr int TILE = BN * RB;
  constexpr int COPIES = TILE / 1024 / NW;  // per wave, K or V
  constexpr int RPC = 1024 / RB;
  constexpr int DB = DT / 32;
  constexpr int KSTEPS = DT / 16;
  static_assert(COPIES >= 1 && COPIES * NW * 1024 == TILE, "whole copies per wave");
  __shared__ __attribute__((aligned(16))) char smem[4 * TILE];  // K, V slots 0; K, V slots 1

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;

  // an XCD (block id mod 8) takes neighbouring query tiles of the same heads: they share keys in its L2
  const int total = p.n_qt * p.batch * p.heads, per = (total + 7) / 8;
  const int lin = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (lin >= total) return;
  const int bh = lin / p.n_qt, qt = p.n_qt - 1 - lin % p.n_qt;
  const int b = bh / p.heads, h = bh % p.heads, kvh = h / p.group;

  const int q0 = qt * (32 * NW);
  const int shift = p.k_len - p.q_len;
  const int row = q0 + wave * 32 + (lane & 31);
  const int pos = shift + row;
  const int w_lo = shift + q0 + wave * 32, w_hi = w_lo + 31;                    // positions of the wave's rows
  const TileList<BN> tiles(p, shift + q0, min(shift + q0 + 32 * NW - 1, p.k_len - 1));

  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + kvh * p.ks[1];
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + kvh * p.vs[1];
  const uint8_t* kvb = KMASK ? p.kv + b * p.kvs : nullptr;
  const uint32_t lds0 = (uint32_t)(size_t)(lds_char*)smem;
  const int last_chunk = p.hd / 8 - 1;

  // Lane l of copy c fills physical chunk l % CPR of row c * RPC + l / CPR with the logical chunk
  // that the swizzle keeps there.  Rows past the keys re-read the last one and chunks past head_dim
  // the last one: their scores are masked, their columns meet zeros of Q or are not stored.
  // A lane's row and chunk never change: their address is kept, and only the tile's is added (a
  // 64-bit product per copy and lane was a fifth of the loop's vector instructions).
  const T *kp[COPIES], *vp[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    const int r = (wave * COPIES + i) * RPC + lane / CPR, phys = lane % CPR;
    kp[i] = kb + r * p.ks[2] + min((swz_off<RB>(r, phys) - r * RB) >> 4, last_chunk) * 8;
    vp[i] = vb + r * p.vs[2] + min(phys ^ vswz<RB>(r), last_chunk) * 8;
  }
  auto copy = [&](int t, uint32_t dst) {
    const int k0 = tiles.key(t);
    const int64_t ko = k0 * p.ks[2], vo = k0 * p.vs[2];
    if (k0 + BN <= p.k_len) {
#pragma unroll
      for (int i = 0; i < COPIES; ++i) dma16(kp[i] + ko, dst + (wave * COPIES + i) * 1024);
#pragma unroll
      for (int i = 0; i < COPIES; ++i) dma16(vp[i] + vo, dst + TILE + (wave * COPIES + i) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int r = (wave * COPIES + i) * RPC + lane / CPR, back = max(k0 + r - (p.k_len - 1), 0);
        dma16(kp[i] + ko - back * p.ks[2], dst + (wave * COPIES + i) * 1024);
        dma16(vp[i] + vo - back * p.vs[2], dst + TILE + (wave * COPIES + i) * 1024);
      }
    }
  };

  x8 qf[KSTEPS];
  {
    const T* qr = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + (int64_t)min(row, p.q_len - 1) * p.qs[2];
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      const int d = 16 * kk + 8 * g;
      qf[kk] = x8{};
      if (d < p.hd) qf[kk] = *reinterpret_cast<const x8*>(qr + d);
    }
  }
  int v_rd[2][DB];  // transposed V reads, as attend_one_tile
  {
    const int tq = lane >> 4, ts = lane & 15;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int vr = 8 * r + 4 * (tq >> 1) + (ts >> 2);
        const int col = 32 * d + 16 * (tq & 1) + 4 * (ts & 3);
        v_rd[r][d] = vr * RB + (((col >> 3) ^ vswz<RB>(vr)) << 4) + (col & 7) * 2;
      }
  }

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float cs = p.scales[0];

  copy(0, lds0);
  for (int t = 0; t < tiles.n; ++t) {
    const int k0 = tiles.key(t);
    char* ks_ = smem + (t & 1) * 2 * TILE;
    char* vs_ = ks_ + TILE;
    uint64_t bits = ~0ull;
    if (KMASK) {
      const int key = k0 + lane;
      bits = __ballot(lane < BN && key < p.k_len && kvb[min(key, p.k_len - 1)] != 0);
    }
    wait_vmcnt<0>();
    if (KMASK && bits != ~0ull >> (64 - BN)) {
      // whatever lies in rows that are not valid times a weight of 0 must be 0
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int c = wave * COPIES + i;
        if (!((bits >> (c * RPC + lane / CPR)) & 1)) *reinterpret_cast<u32x4*>(vs_ + c * 1024 + lane * 16) = u32x4{};
      }
      wait_lds_reads();
    }
    lds_barrier();
    if (t + 1 < tiles.n) copy(t + 1, lds0 + ((t + 1) & 1) * 2 * TILE);
    // nothing of this tile for any of the wave's rows, or no rows (1024 heads of 64, 200 rows: 69.6 -> 63.1 us)
    if (w_lo >= p.k_len || k0 > w_hi || (k0 + BN - 1 <= w_lo - p.window && k0 >= p.sinks)) continue;

    // the products ahead of another wave's exponentials: 588 -> 568 us at head_dim 128
    f32x16 s[NB];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
      for (int kb2 = 0; kb2 < NB; ++kb2) {
        const x8 kf = *reinterpret_cast<const x8*>(ks_ + swz_off<RB>(kb2 * 32 + (lane & 31), 2 * kk + g));
        s[kb2] = Elem<T>::mfma32(kf, qf[kk], kk == 0 ? f32x16{} : s[kb2]);
      }
    __builtin_amdgcn_s_setprio(0);
    const bool whole = k0 + BN - 1 <= w_lo && (k0 > w_hi - p.window || k0 + BN <= p.sinks);
    if (KMASK || !whole) {
      const uint64_t kbits = bits >> (4 * g);
#pragma unroll
      for (int e = 0; e < 16 * NB; ++e) {
        const int j = (e >> 4) * 32 + 8 * ((e & 15) >> 2) + (e & 3), key = k0 + j + 4 * g;
        const bool see = key <= pos && (key > pos - p.window || key < p.sinks) && (!KMASK || ((kbits >> j) & 1));
        if (!see) s[e >> 4][e & 15] = -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16 * NB; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
    const float m_tile = weight_ref<T, 7>(pair_max(mx), p.scales);
    if (__ballot(m_tile > m_run + 8.f) != 0ull) {
      const float m_new = fmaxf(m_run, m_tile);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    x8 pf[2 * NB];
#pragma unroll
    for (int e = 0; e < 16 * NB; ++e)
      pf[e >> 3][e & 7] = (T)__builtin_amdgcn_exp2f(fmaf(s[e >> 4][e & 15], cs, -m_use));
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) l_run = Elem<T>::sum8(pf[i], l_run);
#pragma unroll
    for (int c = 0; c < 2 * NB * DB; ++c) {
      const int t16 = c / DB, d = c % DB;
      const lds_char* base = (const lds_char*)(vs_ + t16 * 16 * RB);
      const tr_f16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr_f16x4*)(base + v_rd[0][d]));
      const tr_f16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr_f16x4*)(base + v_rd[1][d]));
      const f16x8 vf = __builtin_shufflevector(__builtin_bit_cast(f16x4, lo4), __builtin_bit_cast(f16x4, hi4), 0, 1, 2,
                                               3, 4, 5, 6, 7);
      acc[d] = Elem<T>::mfma32(__builtin_bit_cast(x8, vf), pf[t16], acc[d]);
    }
  }

  const float l = pair_sum(l_run);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (row < p.q_len) {
    T* orow = reinterpret_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + (int64_t)row * p.os[2];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int dd = d * 32 + 8 * q + 4 * g;
        if (dd < p.hd)
          *reinterpret_cast<x4*>(orow + dd) = x4{(T)(acc[d][4 * q] * inv), (T)(acc[d][4 * q + 1] * inv),
                                                 (T)(acc[d][4 * q + 2] * inv), (T)(acc[d][4 * q + 3] * inv)};
      }
  }
}

// The same rows' keys dealt to the waves of a workgroup (and to several workgroups): for launches with too
// few query rows to fill the chip, whose workgroups of the kernel above would walk their tiles as one serial
// chain each.  32 rows of one head per workgroup, or of a group's heads one after the other; wave w takes
// every NW-th of its tiles of kSplitKeys keys, into K and V slots of its own, so the loop has no barrier: the
// next K is copied when the current one's products are done, the next V after P.V.  At the end the waves'
// (reference, sum, O) are merged in wave order.  Tiles of 32 keys leave room for seven workgroups per CU at
// head_dim 32, four at 64, two at 128 (at 256 one takes 129 KB): 16 heads of 64, 619 rows, window 126 9.0 us, with
// tiles of 64 11.7.  (Two waves of rows per tile, tiles ahead in a second slot: 14.0, and 31 us instead of 38
// where a window of 2048 keys makes the chains long.)
constexpr int kSplitKeys = 32;
template <typename T, int DT, int NW, bool KMASK>
__device__ __forceinline__ void window_split_body(const WindowArgs& p) {
  constexpr int BN = kSplitKeys;
  typedef typename Elem<T>::x8 x8;
  typedef typename Elem<T>::x4 x4;
  constexpr int NB = BN / 32;
  constexpr int RB = DT * 2;
  constexpr int CPR = RB / 16;
  constexpr int TILE = BN * RB;
  constexpr int COPIES = TILE / 1024;
  constexpr int RPC = 1024 / RB;
  constexpr int DB = DT / 32;
  constexpr int KSTEPS = DT / 16;
  constexpr int SLOT = 2 * TILE;
  constexpr int CHUNKS = 4 * DB;  // 4-register pieces of O
  static_assert(CHUNKS * 1024 <= SLOT && CHUNKS % NW == 0, "a wave's O fits its slots, whole pieces per wave");
  __shared__ __attribute__((aligned(16))) char smem[NW * SLOT];
  __shared__ float row_m[NW][32], row_l[NW][32];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;
  // as in window_body, an XCD takes neighbouring blocks
  const int units = p.heads / p.unit, total = p.n_qt * p.batch * units * p.splits, per = (total + 7) / 8;
  int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int split = id % p.splits;
  id /= p.splits;
  const int qt = id % p.n_qt, bu = id / p.n_qt;
  const int b = bu / units, h0 = bu % units * p.unit, kvh = h0 / p.group;

  // several heads make a list only where each has fewer than 32 rows: the block may hold any of them
  const int q0 = p.unit > 1 ? 0 : qt * 32, shift = p.k_len - p.q_len;
  const int in_list = min(qt * 32 + (lane & 31), p.unit * p.q_len - 1), pos = shift + in_list % p.q_len;
  const int w_lo = shift + q0, w_hi = min(w_lo + 31, p.k_len - 1);
  const TileList<BN> tiles(p, w_lo, w_hi);
  const int t_end = min(tiles.n, (split + 1) * p.per_split);
  int t = split * p.per_split + wave;

  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + kvh * p.ks[1];
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + kvh * p.vs[1];
  const uint8_t* kvb = KMASK ? p.kv + b * p.kvs : nullptr;
  char* ks_ = smem + wave * SLOT;
  char* vs_ = ks_ + TILE;
  const uint32_t k_lds = (uint32_t)(size_t)(lds_char*)ks_, v_lds = k_lds + TILE;
  const int last_chunk = p.hd / 8 - 1;

  auto copy = [&](const T* base, int64_t rs, int k0, uint32_t dst, bool is_v) {  // as in window_body
    const T* tile = base + k0 * rs;
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      const int r = c * RPC + lane / CPR, phys = lane % CPR;
      const int chunk = is_v ? phys ^ vswz<RB>(r) : (swz_off<RB>(r, phys) - r * RB) >> 4;
      dma16(tile + min(r, p.k_len - 1 - k0) * rs + min(chunk, last_chunk) * 8, dst + c * 1024);
    }
  };

  x8 qf[KSTEPS];
  {
    const T* qr = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + (h0 + in_list / p.q_len) * p.qs[1] +
                  (in_list % p.q_len) * p.qs[2];
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      const int d = 16 * kk + 8 * g;
      qf[kk] = x8{};
      if (d < p.hd) qf[kk] = *reinterpret_cast<const x8*>(qr + d);
    }
  }
  if (t < t_end) {
    copy(kb, p.ks[2], tiles.key(t), k_lds, false);
    copy(vb, p.vs[2], tiles.key(t), v_lds, true);
  }
  int v_rd[2][DB];  // transposed V reads, as attend_one_tile
  {
    const int tq = lane >> 4, ts = lane & 15;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int vr = 8 * r + 4 * (tq >> 1) + (ts >> 2);
        const int col = 32 * d + 16 * (tq & 1) + 4 * (ts & 3);
        v_rd[r][d] = vr * RB + (((col >> 3) ^ vswz<RB>(vr)) << 4) + (col & 7) * 2;
      }
  }

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float cs = p.scales[0];

  for (; t < t_end; t += NW) {
    const int k0 = tiles.key(t);
    const bool more = t + NW < t_end;
    int byte = 1;
    if (KMASK) byte = lane < BN && k0 + lane < p.k_len ? kvb[k0 + lane] : 0;
    wait_vmcnt<COPIES>();  // all but V's copies (or fewer, if the validity byte went out before): K has landed
    asm volatile("" ::: "memory");
    f32x16 s[NB];
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
      for (int kb2 = 0; kb2 < NB; ++kb2) {
        const x8 kf = *reinterpret_cast<const x8*>(ks_ + swz_off<RB>(kb2 * 32 + (lane & 31), 2 * kk + g));
        s[kb2] = Elem<T>::mfma32(kf, qf[kk], kk == 0 ? f32x16{} : s[kb2]);
      }
    // every K fragment is in registers: the slot may be refilled
    asm volatile("" ::: "memory");
    wait_lds_reads();
    const uint64_t bits = KMASK ? (uint64_t)__ballot(byte != 0) : ~0ull;  // waits for the byte, and so for V
    if (more) copy(kb, p.ks[2], tiles.key(t + NW), k_lds, false);

    const bool whole = k0 + BN - 1 <= w_lo && (k0 > w_lo + 31 - p.window || k0 + BN <= p.sinks);
    if (KMASK || !whole) {
      const uint64_t kbits = bits >> (4 * g);
#pragma unroll
      for (int e = 0; e < 16 * NB; ++e) {
        const int j = (e >> 4) * 32 + 8 * ((e & 15) >> 2) + (e & 3), key = k0 + j + 4 * g;
        const bool see = key <= pos && (key > pos - p.window || key < p.sinks) && (!KMASK || ((kbits >> j) & 1));
        if (!see) s[e >> 4][e & 15] = -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16 * NB; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
    const float m_tile = weight_ref<T, 7>(pair_max(mx), p.scales);
    if (__ballot(m_tile > m_run + 8.f) != 0ull) {
      const float m_new = fmaxf(m_run, m_tile);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    x8 pf[2 * NB];
#pragma unroll
    for (int e = 0; e < 16 * NB; ++e)
      pf[e >> 3][e & 7] = (T)__builtin_amdgcn_exp2f(fmaf(s[e >> 4][e & 15], cs, -m_use));
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) l_run = Elem<T>::sum8(pf[i], l_run);

    if (more) wait_vmcnt<COPIES>();  // all but the next K's copies
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (KMASK && bits != ~0ull >> (64 - BN)) {
      // whatever lies in rows that are not valid times a weight of 0 must be 0
      const uint32_t mine = (uint32_t)bits >> (lane / CPR);
#pragma unroll
      for (int c = 0; c < COPIES; ++c)
        if (!((mine >> (c * RPC)) & 1)) *reinterpret_cast<u32x4*>(vs_ + c * 1024 + lane * 16) = u32x4{};
      wait_lds_reads();
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int c = 0; c < 2 * NB * DB; ++c) {
      const int t16 = c / DB, d = c % DB;
      const lds_char* base = (const lds_char*)(vs_ + t16 * 16 * RB);
      const tr_f16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr_f16x4*)(base + v_rd[0][d]));
      const tr_f16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr_f16x4*)(base + v_rd[1][d]));
      const f16x8 vf = __builtin_shufflevector(__builtin_bit_cast(f16x4, lo4), __builtin_bit_cast(f16x4, hi4), 0, 1, 2,
                                               3, 4, 5, 6, 7);
      acc[d] = Elem<T>::mfma32(__builtin_bit_cast(x8, vf), pf[t16], acc[d]);
    }
    asm volatile("" ::: "memory");
    wait_lds_reads();
    if (more) copy(vb, p.vs[2], tiles.key(t + NW), v_lds, true);
  }

  // ---- merge: a wave writes its O (CHUNKS of 64 lanes x 16 bytes) into its own slots ----
  asm volatile("" ::: "memory");
  l_run = pair_sum(l_run);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const f32x16& o = acc[c / 4];
    const int q = c % 4;
    *reinterpret_cast<f32x4*>(ks_ + c * 1024 + lane * 16) = f32x4{o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]};
  }
  if (g == 0) {
    row_m[wave][lane] = m_run;
    row_l[wave][lane] = l_run;
  }
  __syncthreads();
  float f[NW], m_all = -INFINITY, l_all = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    f[w] = row_m[w][lane & 31];
    m_all = fmaxf(m_all, f[w]);
  }
  const float m_ref = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    f[w] = __builtin_amdgcn_exp2f(f[w] - m_ref);
    l_all = fmaf(f[w], row_l[w][lane & 31], l_all);
  }
  int listed = lane & 31;
  asm volatile("" : "+v"(listed));  // head and row found anew: they need no registers in the loop
  listed += qt * 32;
  if (listed >= p.unit * p.q_len) return;
  const int h = h0 + listed / p.q_len, row = listed % p.q_len;
  const float inv = l_all == 0.f ? 0.f : 1.0f / l_all;
  T* orow = reinterpret_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + row * p.os[2];
  const int64_t part = (((int64_t)b * p.heads + h) * p.q_len + row) * p.splits + split;
  if (p.splits > 1 && wave == 0 && g == 0) {
    p.stats[2 * part] = m_all;
    p.stats[2 * part + 1] = l_all;
  }
#pragma unroll
  for (int c0 = 0; c0 < CHUNKS; c0 += NW) {
    const int c = c0 + wave, dd = (c / 4) * 32 + 8 * (c % 4) + 4 * g;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(smem + w * SLOT + c * 1024 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f[w], v[e], o[e]);
    }
    if (dd >= p.hd) continue;
    if (p.splits > 1) *reinterpret_cast<f32x4*>(p.part + part * p.hd + dd) = o;
    else *reinterpret_cast<x4*>(orow + dd) = x4{(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
  }
}

template <typename T, int DT, int NW, bool KMASK>
__global__ __launch_bounds__(NW * 64, DT <= 128 ? 2 : 1) void window_split_kernel(WindowArgs p) {
  window_split_body<T, DT, NW, KMASK>(p);
}

template <typename T, int DT, int BN, int NW, bool KMASK>
__global__ __launch_bounds__(NW * 64, DT <= 128 ? 2 : 1) void window_attn_kernel(WindowArgs p) {
  window_body<T, DT, BN, NW, KMASK>(p);
}

constexpr int kWindowWaves = 4;

// Which kernel; for window_split_kernel the heads whose rows make one list, its blocks of 32 rows, and over how
// many workgroups a block's keys are dealt.
struct WindowPlan {
  bool split;
  int64_t unit, blocks;
  int64_t splits, per_split;
};
WindowPlan window_plan(int64_t bh, int64_t group, int64_t q_len, int64_t k_len, int64_t window, int64_t sinks,
                       int64_t hd, bool batch_invariant) {
  // Workgroups of 128 rows fill the chip from one per CU on; two at head_dim 256 (one wave per SIMD), and three to
  // two CUs where a quarter of their waves has no rows and the tiles are short: head_dim 64 and 64 rows, window 512,
  // us in blocks of 32 rows and of 128: 272 heads 15.1, 18.7; 384 14.0, 18.6; 512 21.2, 20.0.  Up to 32 rows a head
  // blocks of 32 win however many heads there are (1024 heads of 128 in groups of 4, window 512: 31, 38; of 256 89,
  // 119), or come close (320 heads of 128, window 2048: 80, 76).
  const int64_t wide = bh * ((q_len + 127) / 128), full = hd > 128 ? 512 : hd <= 64 && q_len <= 96 ? 384 : 256;
  const bool few = q_len <= 32;
  if (!few && (batch_invariant || wide > full)) return {false, 1, wide, 1, 0};
  // Fewer than 32 rows a head: those of a group, which read the same keys, fill the blocks (9 x 32 heads in groups
  // of 4, 8 rows, 3487 keys, head_dim 80: 24 us, a workgroup per head 98).
  const int64_t unit = q_len < 32 && group < (1 << 26) ? group : 1, blocks = bh / unit * ((unit * q_len + 31) / 32);
  int64_t keys = window + 31 + sinks;
  if (keys > k_len) keys = k_len;
  // the sinks and the windows may begin and end inside tiles
  const int64_t tiles = (keys + kSplitKeys - 1) / kSplitKeys + 2;
  if (batch_invariant) return {true, unit, blocks, 1, tiles};
  // A block's keys go to several workgroups only up to one workgroup per CU (8192 rows to be joined at most),
  // in shares of three tiles a wave or more: past that the launch that joins them costs more (10 x 2 heads of
  // 128, 735 rows: whole 20 us, in two 38; 3 heads of 64, 923 rows, window 2920: 18 us in eight shares, 34 whole).
  const int64_t want = blocks < 256 ? 256 / blocks : 1;
  int64_t per = (tiles + want - 1) / want;
  per = (per + kWindowWaves - 1) / kWindowWaves * kWindowWaves;
  if (per < 3 * kWindowWaves) per = 3 * kWindowWaves;
  return {true, unit, blocks, (tiles + per - 1) / per, per};
}

template <typename T, int DT, int BN>
int launch_window(WindowArgs p, const WindowPlan& plan, hipStream_t st) {
  constexpr int NW = kWindowWaves;
  const char* fn = "tk_window_attn";
  p.unit = (int)plan.unit;
  p.n_qt = (int)(plan.blocks / ((int64_t)p.batch * (p.heads / p.unit)));
  const int64_t total = plan.blocks * plan.splits;
  TK_REQUIRE(total <= kMaxGroups, TK_ERR_UNSUPPORTED, "%s: too many workgroups", fn);
  const dim3 g((unsigned)((total + 7) / 8 * 8)), blk(NW * 64);
  if (!plan.split) {
    if (p.kv) hipLaunchKernelGGL((window_attn_kernel<T, DT, BN, NW, true>), g, blk, 0, st, p);
    else hipLaunchKernelGGL((window_attn_kernel<T, DT, BN, NW, false>), g, blk, 0, st, p);
    return check_launch(fn);
  }
  if (p.kv) hipLaunchKernelGGL((window_split_kernel<T, DT, kWindowWaves, true>), g, blk, 0, st, p);
  else hipLaunchKernelGGL((window_split_kernel<T, DT, kWindowWaves, false>), g, blk, 0, st, p);
  const int rc = check_launch(fn);
  if (rc != TK_OK || p.splits == 1) return rc;
  JoinArgs j{};
  j.part = p.part;
  j.stats = p.stats;
  j.o = p.o;
  for (int i = 0; i < 3; ++i) j.os[i] = p.os[i];
  j.heads = p.heads;
  j.q_len = p.q_len;
  j.hd = p.hd;
  j.splits = p.splits;
  j.rows = (int64_t)p.batch * p.heads * p.q_len;
  return launch_join<T>(fn, j, false, st);
}

template <typename T>
int dispatch_window(const WindowArgs& p, const WindowPlan& plan, hipStream_t st) {
  if (p.hd <= 32) return launch_window<T, 32, 64>(p, plan, st);
  if (p.hd <= 64) return launch_window<T, 64, 64>(p, plan, st);
  if (p.hd <= 128) return launch_window<T, 128, 64>(p, plan, st);
  return launch_window<T, 256, 32>(p, plan, st);
}

}  // namespace
}  // namespace tk

using namespace tk;

namespace {

int check_window_shape(const char* fn, int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_len, int64_t k_len,
                       int64_t head_dim, int64_t window, int64_t sinks) {
  TK_REQUIRE(batch >= 0 && heads >= 0 && kv_heads >= 0 && q_len >= 0 && head_dim >= 0 && sinks >= 0 &&
                 batch < (1ll << 31) && heads < (1ll << 31) && kv_heads < (1ll << 31),
             TK_ERR_ARG, "%s: size out of range", fn);
  TK_REQUIRE(q_len <= k_len && k_len < (1ll << 30), TK_ERR_ARG, "%s: q_len=%lld, k_len=%lld: at most k_len queries", fn,
             (long long)q_len, (long long)k_len);
  TK_REQUIRE(window >= 1, TK_ERR_ARG, "%s: window=%lld < 1", fn, (long long)window);
  TK_REQUIRE(kv_heads == 0 ? heads == 0 : heads % kv_heads == 0, TK_ERR_ARG,
             "%s: heads=%lld is no multiple of kv_heads=%lld", fn, (long long)heads, (long long)kv_heads);
  TK_REQUIRE(head_dim <= 256 && head_dim % 8 == 0, TK_ERR_UNSUPPORTED,
             "%s: head_dim=%lld is no multiple of 8 up to 256", fn, (long long)head_dim);
  TK_REQUIRE(batch * heads < (1ll << 31), TK_ERR_UNSUPPORTED, "%s: too many heads in all", fn);
  return TK_OK;
}

// Past every key a window changes nothing, nor do sinks; kept small enough for sums of positions.
int64_t at_most(int64_t x, int64_t k_len) { return x < k_len ? x : k_len; }

int64_t window_workspace(const WindowPlan& plan, int64_t rows, int64_t head_dim) {
  return plan.splits == 1 ? 0 : rows * plan.splits * (head_dim + 2) * (int64_t)sizeof(float);
}

}  // namespace

extern "C" int64_t tk_window_attn_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_len,
                                            int64_t k_len, int64_t head_dim, int64_t window, int64_t sinks,
                                            int batch_invariant) {
  const int rc = check_window_shape("tk_window_attn_workspace", batch, heads, kv_heads, q_len, k_len, head_dim, window,
                                    sinks);
  if (rc != TK_OK) return rc;
  if (batch == 0 || heads == 0 || q_len == 0) return 0;
  return window_workspace(window_plan(batch * heads, heads / kv_heads, q_len, k_len, at_most(window, k_len),
                                      at_most(sinks, k_len), head_dim, batch_invariant != 0),
                          batch * heads * q_len, head_dim);
}

extern "C" int tk_window_attn(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                              const void* v, const int64_t* v_strides, void* out, const int64_t* o_strides, int dtype,
                              int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_len, int64_t k_len,
                              int64_t head_dim, float scale, int64_t window, int64_t sinks, const uint8_t* key_valid,
                              int64_t key_valid_stride, int batch_invariant, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* fn = "tk_window_attn";
  TK_REQUIRE(dtype == TK_F16 || dtype == TK_BF16, TK_ERR_ARG, "%s: dtype %d is not TK_F16 or TK_BF16", fn, dtype);
  const int rc = check_window_shape(fn, batch, heads, kv_heads, q_len, k_len, head_dim, window, sinks);
  if (rc != TK_OK) return rc;
  TK_REQUIRE(scale > 0.f && scale <= kMaxScale, TK_ERR_ARG, "%s: scale must be positive and at most 2.3e38", fn);
  if (batch == 0 || heads == 0 || q_len == 0 || head_dim == 0) return TK_OK;
  TK_REQUIRE(q && k && v && out && q_strides && k_strides && v_strides && o_strides, TK_ERR_ARG, "%s: null pointer", fn);
  TK_REQUIRE(key_valid == nullptr || key_valid_stride >= k_len, TK_ERR_ARG, "%s: key_valid_stride=%lld < k_len", fn,
             (long long)key_valid_stride);
  auto al = [](const void* ptr, uintptr_t a) { return ((uintptr_t)ptr % a) == 0; };
  bool vecs = al(q, 16) && al(k, 16) && al(v, 16) && al(out, 8);
  WindowArgs p{};
  for (int i = 0; i < 3; ++i) {
    vecs = vecs && q_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0 && o_strides[i] % 4 == 0;
    p.qs[i] = q_strides[i];
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
    p.os[i] = o_strides[i];
  }
  TK_REQUIRE(vecs, TK_ERR_UNSUPPORTED, "%s: rows of q, k, v must be 16-byte aligned, of out 8-byte", fn);
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = out;
  p.kv = key_valid;
  p.kvs = key_valid_stride;
  p.batch = (int)batch;
  p.heads = (int)heads;
  p.group = (int)(heads / kv_heads);
  p.q_len = (int)q_len;
  p.k_len = (int)k_len;
  p.hd = (int)head_dim;
  p.window = (int)at_most(window, k_len);
  p.sinks = (int)at_most(sinks, k_len);
  set_scales(p.scales, scale);
  const WindowPlan plan =
      window_plan(batch * heads, p.group, q_len, k_len, p.window, p.sinks, head_dim, batch_invariant != 0);
  const int64_t rows = batch * heads * q_len, need = window_workspace(plan, rows, head_dim);
  TK_REQUIRE(need == 0 || (workspace && al(workspace, 16) && workspace_bytes >= need), TK_ERR_ARG,
             "%s: workspace of %lld bytes, 16-byte aligned, needed", fn, (long long)need);
  p.splits = (int)plan.splits;
  p.per_split = (int)plan.per_split;
  p.part = reinterpret_cast<float*>(workspace);
  p.stats = need ? p.part + rows * plan.splits * head_dim : nullptr;
  return dtype == TK_F16 ? dispatch_window<f16>(p, plan, as_stream(stream))
                         : dispatch_window<bf16>(p, plan, as_stream(stream));
}
