// A paged key/value cache: the write of new tokens, and the bookkeeping of its pages.
//
// A cache is k and v pages [layers][pages][kv_heads][page_size][head_dim], and three int32
// arrays on the device: table [rows][table_width] (a sequence's pages in order), lengths [rows]
// and refs [pages] (how many sequences hold a page; a page is free at refs <= 0).  Sequence b of
// n tokens holds the first ceil(n / page_size) entries of its row; the others mean nothing.
//
// Everything here is decided on the device, so a captured graph can reserve, fork and free
// without the host.  An operation that cannot be done whole changes nothing and says so in
// `status` (below).  Free pages are taken from the lowest id on and nothing depends on the
// order in which workgroups run, so results are the same in every run.
//
// Bounds: the copies by HBM, every moved row read and written once (append of 32768 rows of 16 heads of
// 128 5.3 TB/s, compaction of 64-row pages 5 TB/s); the plans, one workgroup that scans refs 8192 pages at a
// time, by latency (3 to 6 us).
#include "tk_elem.hpp"

namespace tk {
namespace {

constexpr int kPlan = 1024;            // threads of a plan
constexpr int kPlanWaves = kPlan / 64;
constexpr int kScan = 8;               // pages per thread and step of a scan over refs

// status: 0 done, > 0 pages that were missing, kBadRows an entry that cannot be taken
constexpr int kBadRows = -1;

// ------------------------------------------------------------- append --

struct AppendArgs {
  const char* k;
  const char* v;
  char* kp;
  char* vp;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* added;          // nullable: n of every sequence
  const int32_t* status;         // nullable: of the call that made room; nothing is written where it is not 0
  int64_t ks[3], vs[3];          // bytes, {b, token, head}
  int64_t kps[3], vps[3];        // bytes, {page, head, row}
  int64_t table_stride;
  int n, kv_heads, vecs, pages, page_shift, table_width, blocks;  // vecs: 16-byte vectors per row
};

__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs p) {
  const int b = blockIdx.x / p.blocks;
  const int item = (blockIdx.x % p.blocks) * 256 + threadIdx.x;
  const int x = item % p.vecs, r = item / p.vecs;
  const int h = r % p.kv_heads, i = r / p.kv_heads;
  const int n = p.added ? min(p.added[b], p.n) : p.n;
  // a refused reservation left lengths as they were: the rows would land on the newest tokens that are there
  if (i >= n || (p.status && *p.status != 0)) return;
  const int64_t pos = (int64_t)p.lengths[b] - n + i;
  if (pos < 0 || (pos >> p.page_shift) >= p.table_width) return;
  const int page = p.table[b * p.table_stride + (pos >> p.page_shift)];
  if ((uint32_t)page >= (uint32_t)p.pages) return;
  const int64_t row = pos & ((1 << p.page_shift) - 1);
  const u32x4 kx = *reinterpret_cast<const u32x4*>(p.k + b * p.ks[0] + i * p.ks[1] + h * p.ks[2] + 16 * x);
  const u32x4 vx = *reinterpret_cast<const u32x4*>(p.v + b * p.vs[0] + i * p.vs[1] + h * p.vs[2] + 16 * x);
  *reinterpret_cast<u32x4*>(p.kp + page * p.kps[0] + h * p.kps[1] + row * p.kps[2] + 16 * x) = kx;
  *reinterpret_cast<u32x4*>(p.vp + page * p.vps[0] + h * p.vps[1] + row * p.vps[2] + 16 * x) = vx;
}

// -------------------------------------------------------------- plans --

struct CacheArgs {
  char* k;
  char* v;
  int64_t ks[4], vs[4];  // bytes, {layer, page, head, row}
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int64_t table_stride;
  int rows, table_width, pages, page_shift, layers, kv_heads, vecs;
  const int32_t* first;   // reserve: tokens to add; fork: parents; free: rows
  const int32_t* second;  // fork: children
  int n;                  // entries of first
  int32_t* status;
  int32_t* work;
};

constexpr int kFresh = 4096;  // new pages that a plan keeps in LDS; more go through its workspace

struct PlanLds {
  int wave[kPlanWaves];
  int flag;
  int32_t fresh[kFresh];
};

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Exclusive sum over the workgroup's threads; total: the sum of all.
__device__ __forceinline__ int plan_scan(int x, PlanLds& lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 63) lds.wave[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    before += w < wave ? lds.wave[w] : 0;
    total += lds.wave[w];
  }
  __syncthreads();
  return before + incl - x;
}

// A step's refs: thread (wave, lane) holds those of pages base + 512 wave + 64 j + lane.
typedef int PlanRefs[kScan];
__device__ __forceinline__ void load_refs(const int32_t* refs, int pages, int base, PlanRefs& r) {
  const int at = base + (int)(threadIdx.x >> 6) * 64 * kScan + (int)(threadIdx.x & 63);
#pragma unroll
  for (int j = 0; j < kScan; ++j) r[j] = at + 64 * j < pages ? refs[at + 64 * j] : 0;
}

// The pages that `take(page, refs)` picks, in ascending order, into list; stops after a step in
// which `want` were reached.  Returns how many were found (at least min(want, all)).  r: the first
// step's refs, which the caller loads ahead of what it does before (their latency is 2 us on a chip whose
// other XCDs wrote them last).
template <typename Take>
__device__ __forceinline__ int plan_collect(const int32_t* refs, int pages, int want, int32_t* list, int room,
                                            PlanLds& lds, PlanRefs& r, Take take) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int found = 0;
  for (int base = 0; base < pages && found < want; base += kPlan * kScan) {
    const int at = base + wave * 64 * kScan + lane;
    uint64_t mask[kScan];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kScan; ++j) {
      mask[j] = __ballot(at + 64 * j < pages && take(at + 64 * j, r[j]));
      mine += __popcll(mask[j]);
    }
    if (base + kPlan * kScan < pages) load_refs(refs, pages, base + kPlan * kScan, r);
    if (lane == 0) lds.wave[wave] = mine;
    __syncthreads();
    int rank = found;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      rank += w < wave ? lds.wave[w] : 0;
      found += lds.wave[w];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kScan; ++j) {
      const int slot = rank + lanes_below(mask[j]);
      if (((mask[j] >> lane) & 1) && slot < room) list[slot] = at + 64 * j;
      rank += __popcll(mask[j]);
    }
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ int pages_of(int tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

// What row b needs, and where its new pages start in the list of all.
struct ReserveRow {
  int have, need, from, len;  // len: the new length, or -1
};
__device__ __forceinline__ ReserveRow reserve_row(const CacheArgs& p, int b, int before, PlanLds& lds, int& total) {
  const int most = p.table_width << p.page_shift;
  ReserveRow r = {0, 0, 0, 0};
  if (b < p.rows) {
    const int len = p.lengths[b], add = p.first[b];
    if (len < 0 || add < 0 || len > most || add > most - len) {
      lds.flag = 1;
    } else {
      r.have = pages_of(len, p.page_shift);
      r.need = pages_of(len + add, p.page_shift) - r.have;
      r.len = len + add;
    }
  }
  r.from = before + plan_scan(r.need, lds, total);
  return r;
}

// work: [pages] free pages.
__device__ __forceinline__ void reserve_body(const CacheArgs& p) {
  __shared__ PlanLds lds;
  const int lane = threadIdx.x & 63;
  PlanRefs refs;
  load_refs(p.refs, p.pages, 0, refs);
  if (threadIdx.x == 0) lds.flag = 0;
  __syncthreads();
  int total = 0;
  ReserveRow row = {};  // of the last step: with up to kPlan rows it need not be found again
  for (int base = 0; base < p.rows; base += kPlan) {
    int sum;
    row = reserve_row(p, base + (int)threadIdx.x, total, lds, sum);
    total += sum;
  }
  if (lds.flag) {
    if (threadIdx.x == 0) *p.status = kBadRows;
    return;
  }
  int32_t* fresh = total <= kFresh ? lds.fresh : p.work;
  const int found = plan_collect(p.refs, p.pages, total, fresh, total, lds, refs,
                                 [](int, int r) { return r <= 0; });
  if (threadIdx.x == 0) *p.status = max(0, total - found);
  if (found < total) return;
  int before = 0;
  for (int base = 0; base < p.rows; base += kPlan) {
    const int b = base + (int)threadIdx.x;
    if (p.rows > kPlan) {
      int sum;
      row = reserve_row(p, b, before, lds, sum);
      before += sum;
    }
    if (b < p.rows) {
      p.lengths[b] = row.len;
      if (row.need == 1) {
        const int page = fresh[row.from];
        p.table[b * p.table_stride + row.have] = page;
        p.refs[page] = 1;
      }
    }
    // rows that need more (a prompt's): the whole wave for each
    for (uint64_t many = __ballot(row.need > 1); many; many &= many - 1) {
      const int src = __builtin_ctzll(many);
      const int rb = __shfl(b, src), rh = __shfl(row.have, src), rn = __shfl(row.need, src), rf = __shfl(row.from, src);
      for (int i = lane; i < rn; i += 64) {
        const int page = fresh[rf + i];
        p.table[rb * p.table_stride + rh + i] = page;
        p.refs[page] = 1;
      }
    }
  }
}

__global__ __launch_bounds__(kPlan) void cache_reserve_kernel(CacheArgs p) { reserve_body(p); }

// work: [n] parents' lengths, [n] fresh pages, then [pages] free pages.
struct ForkWork {
  int32_t *len, *fresh, *free;
};
__device__ __forceinline__ ForkWork fork_work(const CacheArgs& p) {
  return {p.work, p.work + p.n, p.work + 2 * (int64_t)p.n};
}

constexpr int kForkRows = 1 << 18;  // rows of a table that forks: a bit each in LDS

__device__ __forceinline__ void fork_plan_body(const CacheArgs& p) {
  __shared__ PlanLds lds;
  __shared__ uint32_t seen[kForkRows / 32];  // rows that are children already
  const ForkWork w = fork_work(p);
  const int most = p.table_width << p.page_shift;
  PlanRefs refs;
  load_refs(p.refs, p.pages, 0, refs);
  if (threadIdx.x == 0) lds.flag = 0;
  for (int i = threadIdx.x; i < (p.rows + 31) / 32; i += kPlan) seen[i] = 0;
  __syncthreads();
  int total = 0, rank = -1;  // rank of the last step: with up to kPlan children it need not be kept
  for (int base = 0; base < p.n; base += kPlan) {
    const int i = base + (int)threadIdx.x;
    int need = 0;
    if (i < p.n) {
      const int parent = p.first[i], child = p.second[i];
      int len = -1;
      if ((uint32_t)parent < (uint32_t)p.rows && (uint32_t)child < (uint32_t)p.rows && p.lengths[child] == 0 &&
          !((atomicOr(&seen[child >> 5], 1u << (child & 31)) >> (child & 31)) & 1))
        len = p.lengths[parent];
      if (len < 0 || len > most) lds.flag = 1;
      else need = (len & ((1 << p.page_shift) - 1)) != 0;
      w.len[i] = len;
    }
    int sum;
    const int before = plan_scan(need, lds, sum);
    rank = need ? total + before : -1;
    if (i < p.n && p.n > kPlan) w.fresh[i] = rank;
    total += sum;
  }
  if (lds.flag) {
    if (threadIdx.x == 0) *p.status = kBadRows;
    return;
  }
  int32_t* fresh = total <= kFresh ? lds.fresh : w.free;
  const int found = plan_collect(p.refs, p.pages, total, fresh, total, lds, refs,
                                 [](int, int r) { return r <= 0; });
  if (threadIdx.x == 0) *p.status = max(0, total - found);
  if (found < total) return;
  for (int i = threadIdx.x; i < p.n; i += kPlan) {
    if (p.n > kPlan) rank = w.fresh[i];
    w.fresh[i] = rank >= 0 ? fresh[rank] : -1;
  }
}

__global__ __launch_bounds__(kPlan) void cache_fork_plan_kernel(CacheArgs p) { fork_plan_body(p); }

// One workgroup per child for its table row, and one per child and layer, head for the rows of the begun page.
__global__ __launch_bounds__(256) void cache_fork_kernel(CacheArgs p) {
  if (*p.status != 0) return;
  const ForkWork w = fork_work(p);
  const int parts = 1 + p.layers * p.kv_heads;
  const int i = blockIdx.x / parts, part = blockIdx.x % parts;
  const int len = w.len[i], fresh = w.fresh[i], whole = len >> p.page_shift;
  if (part == 0) {
    const int32_t* from = p.table + p.first[i] * p.table_stride;
    int32_t* to = p.table + p.second[i] * p.table_stride;
    for (int e = threadIdx.x; e < whole; e += 256) {
      const int page = from[e];
      to[e] = page;
      if ((uint32_t)page < (uint32_t)p.pages) atomicAdd(&p.refs[page], 1);
    }
    if (threadIdx.x == 0) {
      if (fresh >= 0) {
        to[whole] = fresh;
        p.refs[fresh] = 1;
      }
      p.lengths[p.second[i]] = len;
    }
    return;
  }
  if (fresh < 0) return;  // (a parent is no child but of an empty row: its entries stand)
  const int src = p.table[p.first[i] * p.table_stride + whole];
  if ((uint32_t)src >= (uint32_t)p.pages) return;
  const int l = (part - 1) / p.kv_heads, h = (part - 1) % p.kv_heads;
  const int items = (len & ((1 << p.page_shift) - 1)) * p.vecs;
  const int64_t kb = l * p.ks[0] + h * p.ks[2], vb = l * p.vs[0] + h * p.vs[2];
  for (int it = threadIdx.x; it < items; it += 256) {
    const int r = it / p.vecs, x = it % p.vecs;
    const int64_t ko = kb + r * p.ks[3] + 16 * x, vo = vb + r * p.vs[3] + 16 * x;
    const u32x4 kx = *reinterpret_cast<const u32x4*>(p.k + src * p.ks[1] + ko);
    const u32x4 vx = *reinterpret_cast<const u32x4*>(p.v + src * p.vs[1] + vo);
    *reinterpret_cast<u32x4*>(p.k + fresh * p.ks[1] + ko) = kx;
    *reinterpret_cast<u32x4*>(p.v + fresh * p.vs[1] + vo) = vx;
  }
}

// One workgroup per listed row; the first to take a row's length empties it.
__global__ __launch_bounds__(256) void cache_free_kernel(CacheArgs p) {
  const int b = p.first[blockIdx.x];
  if ((uint32_t)b >= (uint32_t)p.rows) return;
  __shared__ int taken;
  if (threadIdx.x == 0) taken = atomicExch(&p.lengths[b], 0);
  __syncthreads();
  const int held = min(pages_of(max(taken, 0), p.page_shift), p.table_width);
  int32_t* row = p.table + b * p.table_stride;
  for (int e = threadIdx.x; e < held; e += 256) {
    const int page = row[e];
    row[e] = -1;
    if ((uint32_t)page < (uint32_t)p.pages) atomicSub(&p.refs[page], 1);
  }
}

// work: [1] moves m, [pages] the m holes and the m pages that move into them, [pages] where a page went.
__device__ __forceinline__ void compact_plan_body(const CacheArgs& p) {
  __shared__ PlanLds lds;
  int32_t* list = p.work + 1;
  int32_t* to = list + p.pages;
  int live = 0;
  PlanRefs refs;
  for (int base = (p.pages - 1) / (kPlan * kScan) * (kPlan * kScan); base >= 0; base -= kPlan * kScan) {  // ends with step 0
    load_refs(p.refs, p.pages, base, refs);
#pragma unroll
    for (int j = 0; j < kScan; ++j) live += refs[j] > 0;
  }
  int used;
  plan_scan(live, lds, used);
  for (int i = used + (int)threadIdx.x; i < p.pages; i += kPlan) to[i] = i;
  const int found = plan_collect(p.refs, p.pages, 0x7fffffff, list, p.pages, lds, refs,
                                 [used](int page, int r) { return page < used ? r <= 0 : r > 0; });
  const int m = found / 2;  // as many holes below `used` as live pages above
  for (int i = threadIdx.x; i < m; i += kPlan) {
    const int hole = list[i], page = list[m + i];
    to[page] = hole;
    p.refs[hole] = p.refs[page];
    p.refs[page] = 0;
  }
  if (threadIdx.x == 0) {
    *p.work = m;
    *p.status = used;
  }
}

__global__ __launch_bounds__(kPlan) void cache_compact_plan_kernel(CacheArgs p) { compact_plan_body(p); }

constexpr int kMoveBlocks = 2048;
constexpr int kMoveVecs = 4;  // 16-byte vectors per thread of K and of V

__global__ __launch_bounds__(256) void cache_compact_kernel(CacheArgs p) {
  const int m = *p.work;
  if (m == 0) return;
  const int used = *p.status;
  const int32_t* list = p.work + 1;
  const int32_t* to = list + p.pages;
  for (int b = blockIdx.x; b < p.rows; b += kMoveBlocks) {
    const int held = min(pages_of(max(p.lengths[b], 0), p.page_shift), p.table_width);
    int32_t* row = p.table + b * p.table_stride;
    for (int e = threadIdx.x; e < held; e += 256) {
      const int page = row[e];
      if (page >= used && page < p.pages) row[e] = to[page];
    }
  }
  const int items = (p.kv_heads * p.vecs) << p.page_shift;  // vectors of a page in one layer
  const int chunks = (items + 256 * kMoveVecs - 1) / (256 * kMoveVecs);
  const int64_t units = (int64_t)m * p.layers * chunks;
  for (int64_t u = blockIdx.x; u < units; u += kMoveBlocks) {
    const int ch = (int)(u % chunks);
    const int64_t il = u / chunks;
    const int l = (int)(il % p.layers), i = (int)(il / p.layers);
    const int64_t hole = list[i], page = list[m + i];
    int64_t ko[kMoveVecs], vo[kMoveVecs];
    u32x4 kx[kMoveVecs], vx[kMoveVecs];
#pragma unroll
    for (int j = 0; j < kMoveVecs; ++j) {
      const int it = (ch * kMoveVecs + j) * 256 + (int)threadIdx.x;
      const int x = it % p.vecs, hr = it / p.vecs;
      const int64_t r = hr & ((1 << p.page_shift) - 1), h = hr >> p.page_shift;
      ko[j] = l * p.ks[0] + h * p.ks[2] + r * p.ks[3] + 16 * x;
      vo[j] = l * p.vs[0] + h * p.vs[2] + r * p.vs[3] + 16 * x;
      if (it < items) {
        kx[j] = *reinterpret_cast<const u32x4*>(p.k + page * p.ks[1] + ko[j]);
        vx[j] = *reinterpret_cast<const u32x4*>(p.v + page * p.vs[1] + vo[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kMoveVecs; ++j) {
      if ((ch * kMoveVecs + j) * 256 + (int)threadIdx.x < items) {
        *reinterpret_cast<u32x4*>(p.k + hole * p.ks[1] + ko[j]) = kx[j];
        *reinterpret_cast<u32x4*>(p.v + hole * p.vs[1] + vo[j]) = vx[j];
      }
    }
  }
}

// ------------------------------------------------------------ checks --

bool aligned(const void* ptr, uintptr_t a) { return ((uintptr_t)ptr % a) == 0; }

bool good_page_size(int64_t s) { return s >= 16 && s <= 1024 && (s & (s - 1)) == 0; }

int check_table(const char* fn, const int32_t* table, int64_t stride, int64_t width, int64_t rows,
                const int32_t* lengths, int64_t page_size) {
  TK_REQUIRE(good_page_size(page_size), TK_ERR_UNSUPPORTED, "%s: page_size=%lld is no power of two from 16 to 1024",
             fn, (long long)page_size);
  TK_REQUIRE(rows >= 0 && width >= 0 && rows < (1ll << 24) && width * page_size < (1ll << 30) &&
                 rows * width < (1ll << 31),
             TK_ERR_ARG, "%s: table size out of range", fn);
  TK_REQUIRE(rows <= 1 || stride >= width, TK_ERR_ARG, "%s: table_stride < table_width", fn);
  TK_REQUIRE(rows == 0 || (lengths && (table || width == 0)), TK_ERR_ARG, "%s: null pointer", fn);
  return TK_OK;
}

int check_head_dim(const char* fn, int64_t head_dim) {
  TK_REQUIRE(head_dim >= 0 && head_dim <= 256 && head_dim % 8 == 0, TK_ERR_UNSUPPORTED,
             "%s: head_dim=%lld is no multiple of 8 up to 256", fn, (long long)head_dim);
  return TK_OK;
}

// Strides of 2-byte elements in bytes; rows must stay 16-byte vectors.
int take_strides(const char* fn, int64_t* out, const int64_t* in, int n) {
  for (int i = 0; i < n; ++i) {
    TK_REQUIRE(in[i] % 8 == 0, TK_ERR_UNSUPPORTED, "%s: rows must be 16-byte aligned", fn);
    out[i] = 2 * in[i];
  }
  return TK_OK;
}

int fill_cache(const char* fn, CacheArgs& p, int32_t* table, int64_t table_stride, int64_t table_width, int64_t rows,
               int32_t* lengths, int32_t* refs, int64_t pages, int64_t page_size) {
  const int rc = check_table(fn, table, table_stride, table_width, rows, lengths, page_size);
  if (rc != TK_OK) return rc;
  TK_REQUIRE(pages >= 0 && pages < (1ll << 30) && (refs || pages == 0), TK_ERR_ARG, "%s: bad refs", fn);
  p.table = table;
  p.table_stride = table_stride;
  p.table_width = (int)table_width;
  p.rows = (int)rows;
  p.lengths = lengths;
  p.refs = refs;
  p.pages = (int)pages;
  p.page_shift = __builtin_ctzll((unsigned long long)page_size);
  return TK_OK;
}

int fill_pages(const char* fn, CacheArgs& p, void* k, const int64_t* k_strides, void* v, const int64_t* v_strides,
               int64_t layers, int64_t kv_heads, int64_t head_dim) {
  int rc = check_head_dim(fn, head_dim);
  if (rc != TK_OK) return rc;
  TK_REQUIRE(layers >= 0 && kv_heads >= 0 && layers < (1ll << 16) && kv_heads < (1ll << 16) &&
                 layers * kv_heads < (1ll << 20) && (kv_heads * head_dim << p.page_shift) < (1ll << 30),
             TK_ERR_ARG, "%s: layers, kv_heads or page out of range", fn);
  TK_REQUIRE(k_strides && v_strides, TK_ERR_ARG, "%s: null pointer", fn);
  const bool any = layers > 0 && kv_heads > 0 && head_dim > 0 && p.pages > 0;
  TK_REQUIRE(!any || (k && v), TK_ERR_ARG, "%s: null pointer", fn);
  TK_REQUIRE(aligned(k, 16) && aligned(v, 16), TK_ERR_UNSUPPORTED, "%s: rows must be 16-byte aligned", fn);
  if ((rc = take_strides(fn, p.ks, k_strides, 4)) != TK_OK) return rc;
  if ((rc = take_strides(fn, p.vs, v_strides, 4)) != TK_OK) return rc;
  p.k = (char*)k;
  p.v = (char*)v;
  p.layers = any ? (int)layers : 0;
  p.kv_heads = any ? (int)kv_heads : 0;
  p.vecs = any ? (int)head_dim / 8 : 1;
  return TK_OK;
}

int check_workspace(const char* fn, void* workspace, int64_t bytes, int64_t need) {
  TK_REQUIRE(need == 0 || (workspace && aligned(workspace, 4) && bytes >= need), TK_ERR_ARG,
             "%s: workspace of %lld bytes needed", fn, (long long)need);
  return TK_OK;
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" int64_t tk_cache_workspace(int64_t rows, int64_t pages, int64_t n) {
  TK_REQUIRE(rows >= 0 && pages >= 0 && n >= 0 && rows < (1ll << 24) && pages < (1ll << 30) && n < (1ll << 24),
             TK_ERR_ARG, "tk_cache_workspace: size out of range");
  return 4 * (2 * n + 2 * pages + 1);
}

namespace {

int append(const char* fn, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
           void* k_pages, const int64_t* k_page_strides, void* v_pages, const int64_t* v_page_strides, int64_t batch,
           int64_t n, int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size, const int32_t* table,
           int64_t table_stride, int64_t table_width, const int32_t* lengths, const int32_t* added,
           const int32_t* status, void* stream) {
  int rc = check_table(fn, table, table_stride, table_width, batch, lengths, page_size);
  if (rc != TK_OK) return rc;
  if ((rc = check_head_dim(fn, head_dim)) != TK_OK) return rc;
  TK_REQUIRE(n >= 0 && kv_heads >= 0 && pages >= 0 && n < (1ll << 30) && kv_heads < (1ll << 16) && pages < (1ll << 31),
             TK_ERR_ARG, "%s: size out of range", fn);
  if (batch == 0 || n == 0 || kv_heads == 0 || head_dim == 0 || pages == 0 || table_width == 0) return TK_OK;
  TK_REQUIRE(k && v && k_pages && v_pages && k_strides && v_strides && k_page_strides && v_page_strides, TK_ERR_ARG,
             "%s: null pointer", fn);
  TK_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_pages, 16) && aligned(v_pages, 16), TK_ERR_UNSUPPORTED,
             "%s: rows must be 16-byte aligned", fn);
  AppendArgs p{};
  p.k = (const char*)k;
  p.v = (const char*)v;
  p.kp = (char*)k_pages;
  p.vp = (char*)v_pages;
  p.table = table;
  p.lengths = lengths;
  p.added = added;
  p.status = status;
  if ((rc = take_strides(fn, p.ks, k_strides, 3)) != TK_OK || (rc = take_strides(fn, p.vs, v_strides, 3)) != TK_OK ||
      (rc = take_strides(fn, p.kps, k_page_strides, 3)) != TK_OK ||
      (rc = take_strides(fn, p.vps, v_page_strides, 3)) != TK_OK)
    return rc;
  p.table_stride = table_stride;
  p.n = (int)n;
  p.kv_heads = (int)kv_heads;
  p.vecs = (int)head_dim / 8;
  p.pages = (int)pages;
  p.page_shift = __builtin_ctzll((unsigned long long)page_size);
  p.table_width = (int)table_width;
  const int64_t items = n * kv_heads * p.vecs, blocks = (items + 255) / 256;
  TK_REQUIRE(items < (1ll << 31) - 256 && blocks * batch <= kMaxGroups, TK_ERR_UNSUPPORTED, "%s: too many rows", fn);
  p.blocks = (int)blocks;
  hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)(blocks * batch)), dim3(256), 0, as_stream(stream), p);
  return check_launch(fn);
}

}  // namespace

extern "C" int tk_cache_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                               void* k_pages, const int64_t* k_page_strides, void* v_pages,
                               const int64_t* v_page_strides, int64_t batch, int64_t n, int64_t kv_heads,
                               int64_t head_dim, int64_t pages, int64_t page_size, const int32_t* table,
                               int64_t table_stride, int64_t table_width, const int32_t* lengths,
                               const int32_t* added, void* stream) {
  return append("tk_cache_append", k, k_strides, v, v_strides, k_pages, k_page_strides, v_pages, v_page_strides, batch,
                n, kv_heads, head_dim, pages, page_size, table, table_stride, table_width, lengths, added, nullptr,
                stream);
}

extern "C" int tk_cache_append_reserved(const void* k, const int64_t* k_strides, const void* v,
                                        const int64_t* v_strides, void* k_pages, const int64_t* k_page_strides,
                                        void* v_pages, const int64_t* v_page_strides, int64_t batch, int64_t n,
                                        int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size,
                                        const int32_t* table, int64_t table_stride, int64_t table_width,
                                        const int32_t* lengths, const int32_t* added, const int32_t* status,
                                        void* stream) {
  const char* fn = "tk_cache_append_reserved";
  TK_REQUIRE(status, TK_ERR_ARG, "%s: null pointer", fn);
  return append(fn, k, k_strides, v, v_strides, k_pages, k_page_strides, v_pages, v_page_strides, batch, n, kv_heads,
                head_dim, pages, page_size, table, table_stride, table_width, lengths, added, status, stream);
}

extern "C" int tk_cache_reserve(int32_t* table, int64_t table_stride, int64_t table_width, int64_t rows,
                                int32_t* lengths, int32_t* refs, int64_t pages, int64_t page_size,
                                const int32_t* added, int32_t* status, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  const char* fn = "tk_cache_reserve";
  CacheArgs p{};
  int rc = fill_cache(fn, p, table, table_stride, table_width, rows, lengths, refs, pages, page_size);
  if (rc != TK_OK) return rc;
  TK_REQUIRE(status && (added || rows == 0), TK_ERR_ARG, "%s: null pointer", fn);
  if ((rc = check_workspace(fn, workspace, workspace_bytes, 4 * pages)) != TK_OK) return rc;
  p.first = added;
  p.status = status;
  p.work = (int32_t*)workspace;
  hipLaunchKernelGGL(cache_reserve_kernel, dim3(1), dim3(kPlan), 0, as_stream(stream), p);
  return check_launch(fn);
}

extern "C" int tk_cache_fork(void* k_pages, const int64_t* k_strides, void* v_pages, const int64_t* v_strides,
                             int64_t layers, int64_t kv_heads, int64_t head_dim, int32_t* table, int64_t table_stride,
                             int64_t table_width, int64_t rows, int32_t* lengths, int32_t* refs, int64_t pages,
                             int64_t page_size, const int32_t* parents, const int32_t* children, int64_t n,
                             int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "tk_cache_fork";
  CacheArgs p{};
  int rc = fill_cache(fn, p, table, table_stride, table_width, rows, lengths, refs, pages, page_size);
  if (rc != TK_OK) return rc;
  if ((rc = fill_pages(fn, p, k_pages, k_strides, v_pages, v_strides, layers, kv_heads, head_dim)) != TK_OK) return rc;
  TK_REQUIRE(n >= 0 && n < (1ll << 24) && status && (n == 0 || (parents && children)), TK_ERR_ARG,
             "%s: bad parents or children", fn);
  TK_REQUIRE(rows <= kForkRows, TK_ERR_UNSUPPORTED, "%s: a table of more than %d rows", fn, kForkRows);
  if ((rc = check_workspace(fn, workspace, workspace_bytes, 4 * (2 * n + pages))) != TK_OK) return rc;
  const int64_t grid = n * (1 + (int64_t)p.layers * p.kv_heads);
  TK_REQUIRE(grid <= kMaxGroups, TK_ERR_UNSUPPORTED, "%s: too many children", fn);
  p.first = parents;
  p.second = children;
  p.n = (int)n;
  p.status = status;
  p.work = (int32_t*)workspace;
  hipLaunchKernelGGL(cache_fork_plan_kernel, dim3(1), dim3(kPlan), 0, as_stream(stream), p);
  if ((rc = check_launch(fn)) != TK_OK || n == 0) return rc;
  hipLaunchKernelGGL(cache_fork_kernel, dim3((unsigned)grid), dim3(256), 0, as_stream(stream), p);
  return check_launch(fn);
}

extern "C" int tk_cache_free(int32_t* table, int64_t table_stride, int64_t table_width, int64_t rows,
                             int32_t* lengths, int32_t* refs, int64_t pages, int64_t page_size, const int32_t* list,
                             int64_t n, void* stream) {
  const char* fn = "tk_cache_free";
  CacheArgs p{};
  const int rc = fill_cache(fn, p, table, table_stride, table_width, rows, lengths, refs, pages, page_size);
  if (rc != TK_OK) return rc;
  TK_REQUIRE(n >= 0 && n <= kMaxGroups && (n == 0 || list), TK_ERR_ARG, "%s: bad list of rows", fn);
  if (n == 0) return TK_OK;
  p.first = list;
  p.n = (int)n;
  hipLaunchKernelGGL(cache_free_kernel, dim3((unsigned)n), dim3(256), 0, as_stream(stream), p);
  return check_launch(fn);
}

extern "C" int tk_cache_compact(void* k_pages, const int64_t* k_strides, void* v_pages, const int64_t* v_strides,
                                int64_t layers, int64_t kv_heads, int64_t head_dim, int32_t* table,
                                int64_t table_stride, int64_t table_width, int64_t rows, const int32_t* lengths,
                                int32_t* refs, int64_t pages, int64_t page_size, int32_t* used, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  const char* fn = "tk_cache_compact";
  CacheArgs p{};
  int rc = fill_cache(fn, p, table, table_stride, table_width, rows, const_cast<int32_t*>(lengths), refs, pages,
                      page_size);
  if (rc != TK_OK) return rc;
  if ((rc = fill_pages(fn, p, k_pages, k_strides, v_pages, v_strides, layers, kv_heads, head_dim)) != TK_OK) return rc;
  TK_REQUIRE(used, TK_ERR_ARG, "%s: null pointer", fn);
  if ((rc = check_workspace(fn, workspace, workspace_bytes, 4 * (1 + 2 * pages))) != TK_OK) return rc;
  p.status = used;
  p.work = (int32_t*)workspace;
  hipLaunchKernelGGL(cache_compact_plan_kernel, dim3(1), dim3(kPlan), 0, as_stream(stream), p);
  if ((rc = check_launch(fn)) != TK_OK) return rc;
  hipLaunchKernelGGL(cache_compact_kernel, dim3(kMoveBlocks), dim3(256), 0, as_stream(stream), p);
  return check_launch(fn);
}
