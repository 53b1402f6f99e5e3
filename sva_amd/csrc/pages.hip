// The pages of a KV cache: rows written and read, pages copied, handed out,
// shared, freed and moved together (pages.h).
//
// Which page belongs to whom is integers on the device: tables [S, M], lengths
// [S] and refs [pages], the number of table entries that name a page (0:
// free).  New pages are always the lowest free ones, in the order of the
// sequences, and counts change by integer atomics: results do not depend on
// the order in which threads run.
#include <algorithm>

#include "capi_internal.h"
#include "pages.h"

using namespace sva;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ rows

struct RowsParams {
  Pages c;
  unsigned char* keys;
  unsigned char* values;
  int64_t kv_bs, kv_hs, kv_rs;  // bytes
  const int64_t* first_rows;
  int64_t n_rows;
  int G, chunks;  // 16-byte chunks of a row
  int es;
  uint32_t blocks;  // of one head's K or V
};

// One 16-byte chunk of a row a thread, a head's rows one after another as they
// lie in the page, `blocks` workgroups for each (sequence, head, K or V).  WRITE: into the pages, else
// out of them (rows without a page read as 0).  A sequence whose first row is
// below 0 has none of them (a first row of -1 says that it was given no room:
// its second token is not to land in row 0).  VEC: rows in memory are whole
// aligned 16-byte words.  Bound by memory where there are many rows (131072 of
// 8 x 128 bf16 written: 195 us, 5.5 TB/s), by the latency of page number and row
// where there are few (32 of 3 x 64: 2.7 us).
template <bool WRITE, bool VEC>
__global__ void __launch_bounds__(256) page_rows_kernel(RowsParams p) {
  const uint32_t y = blockIdx.x / p.blocks;
  const int kv = (int)(y & 1), g = (int)((y >> 1) % (uint32_t)p.G), b = (int)((y >> 1) / (uint32_t)p.G);
  const int64_t first = p.first_rows[b];
  unsigned char* rows = (kv ? p.values : p.keys) + b * p.kv_bs + g * p.kv_hs;
  const int64_t rowb = (int64_t)p.chunks * 16;
  const int64_t inside = (((int64_t)(kv * p.G + g)) << p.c.bits) * rowb;
  const int64_t total = p.n_rows * p.chunks;
  for (int64_t i = (int64_t)(blockIdx.x % p.blocks) * 256 + threadIdx.x; i < total; i += (int64_t)p.blocks * 256) {
    const int64_t t = (uint64_t)i / (uint32_t)p.chunks;
    const int ch = (int)(i - t * p.chunks);
    const uint64_t n = (uint64_t)first + (uint64_t)t, at = n >> p.c.bits;
    const int page = first >= 0 && at < (uint64_t)p.c.max_pages ? page_of(p.c, b, (int)at) : -1;
    if (WRITE && page < 0) continue;
    unsigned char* there = p.c.pool + (int64_t)(page < 0 ? 0 : page) * p.c.page_bytes + inside +
                           (int64_t)(n & ((1u << p.c.bits) - 1)) * rowb + ch * 16;
    unsigned char* here = rows + t * p.kv_rs + ch * 16;
    u32x4 x = {0u, 0u, 0u, 0u};
    if (WRITE) {
      if (VEC) {
        x = *(const u32x4*)here;
      } else if (p.es == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = ((const uint32_t*)here)[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k] = (uint32_t)((const uint16_t*)here)[2 * k] | (uint32_t)((const uint16_t*)here)[2 * k + 1] << 16;
      }
      *(u32x4*)there = x;
    } else {
      if (page >= 0) x = *(const u32x4*)there;
      *(u32x4*)here = x;  // (the host allocates whole rows)
    }
  }
}

// ------------------------------------------------------------------ copies

struct CopyParams {
  unsigned char* pool;
  int64_t pages, page_bytes, layer_bytes;  // distances
  int64_t bytes;                           // of one page, a multiple of 16
  const int32_t* src;
  const int32_t* dst;
  int64_t pairs;
  int pieces;  // workgroups a page
};

constexpr int kPiece = 16384;  // bytes of a page that a workgroup copies at a time

// x: pieces of a page, y: pairs, z: layers.  A wave reads 64 pairs at once and
// goes on to those that are there: lists that are mostly -1 cost a load for 64
// of them.  Bound by memory (983 pages of 64 KB of 8 layers: 199 us, 5.2 TB/s read and
// written).
__global__ void __launch_bounds__(256) pages_copy_kernel(CopyParams p) {
  unsigned char* pool = p.pool + (int64_t)blockIdx.z * p.layer_bytes;
  const int64_t from = (int64_t)blockIdx.x * kPiece + (int64_t)threadIdx.x * 16;
  for (int64_t i0 = blockIdx.y; i0 < p.pairs; i0 += (int64_t)gridDim.y * WAVE) {
    const int64_t i = i0 + (int64_t)lane_id() * gridDim.y;
    int s = -1, d = -1;
    if (i < p.pairs) s = p.src[i], d = p.dst[i];
    uint64_t left = __ballot(s >= 0 && s < p.pages && d >= 0 && d < p.pages && s != d);
    for (; left != 0ull; left &= left - 1) {
      const int at = __builtin_ctzll(left);
      const unsigned char* a = pool + (int64_t)__builtin_amdgcn_readlane(s, at) * p.page_bytes;
      unsigned char* c = pool + (int64_t)__builtin_amdgcn_readlane(d, at) * p.page_bytes;
      u32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (from + 4096 * k < p.bytes) x[k] = *(const u32x4*)(a + from + 4096 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (from + 4096 * k < p.bytes) *(u32x4*)(c + from + 4096 * k) = x[k];
    }
  }
}

// ------------------------------------------------------------------ who holds what

struct HoldParams {
  int32_t* tables;
  int64_t table_stride;
  int64_t* lens;
  int32_t* refs;
  int64_t S, M, pages;
  int bits;
};

SVA_DEV int64_t pages_for(int64_t rows, int bits) { return (rows + (1 << bits) - 1) >> bits; }
SVA_DEV bool is_page(const HoldParams& p, int id) { return id >= 0 && id < p.pages; }

constexpr int HB = 1024;
constexpr int HW = HB / WAVE;

// Inclusive sum over the workgroup's threads in order, and the sum of all.
SVA_DEV int64_t block_upto(int64_t v, int64_t* scratch, int64_t& total) {
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
#pragma unroll
  for (int s = 1; s < WAVE; s <<= 1) {
    const int64_t x = __shfl_up(v, s, WAVE);
    if (lane >= s) v += x;
  }
  __syncthreads();
  if (lane == WAVE - 1) scratch[w] = v;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < HW; ++k) {
    before += k < w ? scratch[k] : 0;
    total += scratch[k];
  }
  return v + before;
}

// 16 waves x 16 x 64 pages from `base` on: this thread's counts (behind the
// end: of the last page).
constexpr int PR = 16;  // pages a thread at a time
SVA_DEV int64_t my_page(int64_t base) { return base + (int64_t)(threadIdx.x / WAVE) * (WAVE * PR) + lane_id(); }
SVA_DEV void load_refs(const int32_t* refs, int64_t pages, int64_t base, int32_t (&r)[PR]) {
#pragma unroll
  for (int k = 0; k < PR; ++k) r[k] = refs[min(my_page(base) + k * WAVE, pages - 1)];
}
// Of these pages, those of which pick(page, refs) says so: got(page, rank) is
// told their ranks from `found` on, which grows by their number.
template <typename Pick, typename Got>
SVA_DEV void rank_chunk(const int32_t (&r)[PR], int64_t pages, int64_t base, int64_t* scratch, int64_t& found, Pick pick,
                        Got got) {
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
  uint64_t mask[PR];
  int count = 0;
#pragma unroll
  for (int k = 0; k < PR; ++k) {
    const int64_t page = my_page(base) + k * WAVE;
    mask[k] = __ballot(page < pages && pick(page, r[k]));
    count += (int)__popcll(mask[k]);
  }
  __syncthreads();
  if (lane == 0) scratch[w] = count;
  __syncthreads();
  int64_t rank = found;
#pragma unroll
  for (int k = 0; k < HW; ++k) {
    rank += k < w ? scratch[k] : 0;
    found += scratch[k];
  }
#pragma unroll
  for (int k = 0; k < PR; ++k) {
    if (mask[k] >> lane & 1ull) got(my_page(base) + k * WAVE, rank + (int)__popcll(mask[k] & ((1ull << lane) - 1)));
    rank += (int)__popcll(mask[k]);
  }
}

// What a sequence asks for: pages up to it (its own among them), the table
// position of its first new one, and the shared page that it leaves (or -1).
struct Ask {
  int64_t upto;
  int32_t begin, leaves;
};

// Up to these sizes what the sequences ask for and get is kept in LDS.
constexpr int64_t kFewSeqs = 1024, kFewPages = 8192;
inline bool reserve_small(int64_t n_seq, int64_t n_pages) { return n_seq <= kFewSeqs && n_pages <= kFewPages; }

// Room for counts[s] more rows behind every sequence, one workgroup: what each
// asks for, in order; the free pages by rank; their way into the tables.  A
// last page that others hold too is left to them where rows are to go into it:
// the pair (it, the new one) is to be copied.  Bound by the latency of its
// steps: the scan of refs, whose first chunk is under way from the start, ends
// with the last page that is wanted (4 sequences of 256 pages 8.5 us, 64 of 384
// 12.3).
template <bool SMALL>
__global__ void __launch_bounds__(HB) pages_reserve_kernel(HoldParams p, const int64_t* counts, int64_t each, Ask* asks,
                                                           int32_t* list, int64_t* first_rows, int32_t* src,
                                                           int32_t* dst) {
  __shared__ int64_t scratch[HW];
  __shared__ Ask lds_asks[SMALL ? kFewSeqs : 1];
  __shared__ int32_t lds_list[SMALL ? kFewPages : 1];
  if (SMALL) asks = lds_asks, list = lds_list;
  const int tid = (int)threadIdx.x;
  int32_t r[PR];
  load_refs(p.refs, p.pages, 0, r);
  int64_t wanted = 0;
  for (int64_t s0 = 0; s0 < p.S; s0 += HB) {
    const int64_t s = s0 + tid;
    Ask a = {0, -1, -1};
    int64_t need = 0;
    if (s < p.S) {
      const int64_t len = p.lens[s], c = counts ? counts[s] : each;
      if (c >= 0 && len >= 0 && len <= (p.M << p.bits) && c <= (p.M << p.bits) - len) {
        const int64_t old = pages_for(len, p.bits);
        a.begin = (int32_t)old;
        if (c > 0 && (len & ((1 << p.bits) - 1)) != 0) {
          const int last = p.tables[s * p.table_stride + old - 1];
          if (is_page(p, last) && p.refs[last] > 1) a.leaves = last, --a.begin;
        }
        need = pages_for(len + c, p.bits) - a.begin;
      }
    }
    int64_t total;
    a.upto = wanted + block_upto(need, scratch, total);
    wanted += total;
    if (s < p.S) asks[s] = a;
  }
  int64_t found = 0;
  for (int64_t base = 0; base < p.pages && found < wanted; base += HB * PR) {
    if (base > 0) load_refs(p.refs, p.pages, base, r);
    rank_chunk(
        r, p.pages, base, scratch, found, [](int64_t, int32_t n) { return n == 0; },
        [&](int64_t page, int64_t rank) {
          if (rank < wanted) list[rank] = (int32_t)page;
        });
  }
  __syncthreads();
  // page r of the list: its sequence by bisection
  for (int64_t r = tid; r < (wanted < found ? wanted : found); r += HB) {
    int64_t lo = 0, hi = p.S - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (asks[mid].upto > r) hi = mid;
      else lo = mid + 1;
    }
    if (asks[lo].upto > found) continue;
    const int64_t before = lo > 0 ? asks[lo - 1].upto : 0;
    p.tables[lo * p.table_stride + asks[lo].begin + (r - before)] = list[r];
    p.refs[list[r]] = 1;
  }
  __syncthreads();
  for (int64_t s = tid; s < p.S; s += HB) {
    const Ask a = asks[s];
    const int64_t before = s > 0 ? asks[s - 1].upto : 0, len = p.lens[s];
    const bool granted = a.begin >= 0 && (a.upto == before || a.upto <= found);
    const bool parts = granted && a.leaves >= 0;
    first_rows[s] = granted ? len : -1;
    src[s] = parts ? a.leaves : -1;
    dst[s] = parts ? list[before] : -1;
    if (parts) atomicSub(p.refs + a.leaves, 1);
    if (granted) p.lens[s] = len + (counts ? counts[s] : each);
  }
}

// Row s of the tables becomes a fork of row sources[s] (-1: of none, it is
// freed; itself or no row: as it is).  All are read before any is written, since
// a source may be replaced itself; the counts follow by integer atomics.
SVA_DEV bool forked(const HoldParams& p, const int64_t* sources, int64_t s, int64_t& from) {
  from = sources[s];
  return from != s && from >= -1 && from < p.S;
}
SVA_DEV int64_t held_by(const HoldParams& p, int64_t s) {
  const int64_t n = pages_for(max(p.lens[s], (int64_t)0), p.bits);
  return n < p.M ? n : p.M;
}

// Entry j of row s: what it becomes (counted), by `next`; whether row s changes.
template <typename Next>
SVA_DEV void fork_entry(const HoldParams& p, const int64_t* sources, int64_t s, int64_t j, Next next) {
  int64_t from;
  if (!forked(p, sources, s, from)) return;
  int id = -1;
  if (from >= 0 && j < held_by(p, from)) id = p.tables[from * p.table_stride + j];
  if (is_page(p, id)) atomicAdd(p.refs + id, 1);
  const int old = j < held_by(p, s) ? p.tables[s * p.table_stride + j] : -1;
  if (is_page(p, old)) atomicSub(p.refs + old, 1);
  next(id, from < 0 ? 0 : p.lens[from]);
}

// Tables of few entries: one workgroup, an entry a thread, the new ones in
// registers meanwhile (4 x 33: 2.9 us, 4.3 in two launches; 64 x 33 as three
// entries a thread 7.5, 6.1).
constexpr int64_t kFewEntries = HB;
__global__ void __launch_bounds__(HB) pages_fork_few_kernel(HoldParams p, const int64_t* sources) {
  const int s = (int)threadIdx.x / (int)p.M, j = (int)threadIdx.x % (int)p.M;
  int id = -1;
  int64_t len = 0;
  bool moved = false;
  if (s < p.S) fork_entry(p, sources, s, j, [&](int page, int64_t n) { id = page, len = n, moved = true; });
  __syncthreads();
  if (!moved) return;
  p.tables[s * p.table_stride + j] = id;
  if (j == 0) p.lens[s] = len;
}

// Others: into `next` first, then back.
__global__ void __launch_bounds__(256) pages_fork_kernel(HoldParams p, const int64_t* sources, int32_t* next,
                                                         int64_t* next_lens) {
  const int64_t s = blockIdx.x, j = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (j >= p.M) return;
  fork_entry(p, sources, s, j, [&](int page, int64_t n) {
    next[s * p.M + j] = page;
    if (j == 0) next_lens[s] = n;
  });
}

__global__ void __launch_bounds__(256) pages_forked_kernel(HoldParams p, const int64_t* sources, const int32_t* next,
                                                           const int64_t* next_lens) {
  const int64_t s = blockIdx.x, j = (int64_t)blockIdx.y * 256 + threadIdx.x;
  int64_t from;
  if (j >= p.M || !forked(p, sources, s, from)) return;
  p.tables[s * p.table_stride + j] = next[s * p.M + j];
  if (j == 0) p.lens[s] = next_lens[s];
}

// The pages in use moved to the front: with U of them, the k-th one in use
// from U on goes to the k-th free one below U.  One workgroup counts, ranks
// and moves the refs; the tables follow, the pages themselves are copied by
// the caller's pairs.  Bound by the latency of the scans (512 pages 9.6 us, 4096
// 10.6).
__global__ void __launch_bounds__(HB) pages_compact_kernel(int32_t* refs, int64_t pages, int32_t* to, int32_t* src,
                                                           int32_t* dst, int64_t n_pairs, int32_t* used) {
  __shared__ int64_t scratch[HW];
  int64_t U = 0, holes = 0, moves = 0;
  int32_t r[PR];
  for (int64_t base = 0; base < pages; base += HB * PR) {
    load_refs(refs, pages, base, r);
    rank_chunk(
        r, pages, base, scratch, U,
        [&](int64_t page, int32_t n) {
          to[page] = (int32_t)page;  // (also of free pages, which a table may still name)
          return n > 0;
        },
        [](int64_t, int64_t) {});
  }
  for (int64_t base = 0; base < pages; base += HB * PR) {
    if (pages > HB * PR) load_refs(refs, pages, base, r);
    if (base < U)
      rank_chunk(
          r, pages, base, scratch, holes, [&](int64_t page, int32_t n) { return page < U && n <= 0; },
          [&](int64_t page, int64_t k) { dst[k] = (int32_t)page; });
    if (base + HB * PR > U)
      rank_chunk(
          r, pages, base, scratch, moves, [&](int64_t page, int32_t n) { return page >= U && n > 0; },
          [&](int64_t page, int64_t k) { src[k] = (int32_t)page; });
  }
  __syncthreads();
  for (int64_t k = threadIdx.x; k < n_pairs; k += HB) {
    if (k < moves) {
      const int a = src[k], b = dst[k];
      to[a] = b;
      refs[b] = refs[a];
      refs[a] = 0;
    } else {
      src[k] = dst[k] = -1;
    }
  }
  if (threadIdx.x == 0) *used = (int32_t)U;
}

__global__ void __launch_bounds__(256) pages_renamed_kernel(int32_t* tables, int64_t table_stride, int64_t M, int64_t pages,
                                                            const int32_t* to, const int32_t* used) {
  const int64_t j = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (j >= M) return;
  int32_t* at = tables + (int64_t)blockIdx.x * table_stride + j;
  const int id = *at;
  if (id < *used || id >= pages) return;
  *at = to[id];
}

HoldParams hold(int32_t* tables, int64_t table_stride, int64_t* lens, int32_t* refs, int64_t n_seq, int64_t max_pages,
                int64_t n_pages, int64_t page_rows) {
  HoldParams p;
  p.tables = tables;
  p.table_stride = table_stride;
  p.lens = lens;
  p.refs = refs;
  p.S = n_seq;
  p.M = max_pages;
  p.pages = n_pages;
  p.bits = page_bits(page_rows);
  return p;
}

// (grids: rows in x, table entries in y)
bool sizes_ok(int64_t n_seq, int64_t max_pages, int64_t n_pages) {
  return n_seq > 0 && max_pages > 0 && n_pages > 0 && n_seq < (1ll << 31) && max_pages <= 65535ll * 256 &&
         n_pages < (1ll << 31);
}

template <bool WRITE>
int rows(const char* name, const void* keys, const void* values, int kv_dtype, int64_t kv_seq_stride,
         int64_t kv_head_stride, int64_t kv_row_stride, int64_t n_seq, int64_t n_rows, int64_t G, int64_t D,
         const int64_t* first_rows, const void* pool, int64_t n_pages, int64_t page_stride, int64_t page_rows,
         const int32_t* tables, int64_t table_stride, int64_t max_pages, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(keys && values && first_rows && pool && tables, "%s: null pointer", name);
  SVA_REQUIRE(n_seq > 0 && n_rows > 0 && G > 0 && n_pages > 0 && max_pages > 0, "%s: bad sizes", name);
  SVA_REQUIRE(kv_dtype >= 0 && kv_dtype <= 2, "%s: bad dtype", name);
  SVA_REQUIRE(D > 0 && D <= 256 && D % 8 == 0, "%s: head_dim %lld is not a multiple of 8 up to 256", name, (long long)D);
  SVA_REQUIRE(page_rows_ok(page_rows), "%s: %lld rows a page are no power of two from 16 to 1024", name,
              (long long)page_rows);
  const int64_t es = kv_dtype == F32 ? 4 : 2;
  SVA_REQUIRE(((uintptr_t)pool & 15u) == 0 && page_stride * es % 16 == 0 && page_stride >= 2 * G * page_rows * D,
              "%s: pages are not 16-byte aligned blocks of 2 x G x rows x head_dim elements", name);
  SVA_REQUIRE(n_pages < (1ll << 31) && max_pages < (1ll << 31) && n_rows < (1ll << 40), "%s: too many pages or rows", name);
  SVA_REQUIRE(n_seq < (1ll << 31) && G < (1ll << 20), "%s: too many sequences or heads", name);
  RowsParams p;
  p.c.pool = (unsigned char*)const_cast<void*>(pool);
  p.c.page_bytes = page_stride * es;
  p.c.pages = n_pages;
  p.c.tables = tables;
  p.c.table_stride = table_stride;
  p.c.max_pages = (int)max_pages;
  p.c.bits = page_bits(page_rows);
  p.keys = (unsigned char*)const_cast<void*>(keys);
  p.values = (unsigned char*)const_cast<void*>(values);
  p.kv_bs = kv_seq_stride * es;
  p.kv_hs = kv_head_stride * es;
  p.kv_rs = kv_row_stride * es;
  p.first_rows = first_rows;
  p.n_rows = n_rows;
  p.G = (int)G;
  p.chunks = (int)(D * es / 16);
  p.es = (int)es;
  const bool vec = (((uintptr_t)keys | (uintptr_t)values) & 15u) == 0 && p.kv_bs % 16 == 0 && p.kv_hs % 16 == 0 &&
                   p.kv_rs % 16 == 0;
  SVA_REQUIRE(WRITE || vec, "%s: outputs are not 16-byte aligned rows", name);
  // (4096 workgroups for a head, fewer where that would be more than a grid holds)
  const int64_t heads = 2 * n_seq * G;
  const int64_t blocks = std::min<int64_t>({(n_rows * p.chunks + 255) / 256, 4096, ((1ll << 31) - 1) / heads});
  SVA_UNSUPPORTED(blocks > 0, "%s: %lld sequences of %lld heads in one call", name, (long long)n_seq, (long long)G);
  p.blocks = (uint32_t)blocks;
  const dim3 grid((unsigned)(blocks * heads));
  if (vec) hipLaunchKernelGGL((page_rows_kernel<WRITE, true>), grid, dim3(256), 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL((page_rows_kernel<WRITE, false>), grid, dim3(256), 0, (hipStream_t)stream, p);
  SVA_CHECK_LAUNCH("page_rows_kernel");
  return SVA_OK;
}

}  // namespace

extern "C" int sva_paged_write(const void* keys, const void* values, int kv_dtype, int64_t kv_seq_stride,
                               int64_t kv_head_stride, int64_t kv_row_stride, int64_t n_seq, int64_t n_rows, int64_t G,
                               int64_t D, const int64_t* first_rows, void* pool, int64_t n_pages, int64_t page_stride,
                               int64_t page_rows, const int32_t* tables, int64_t table_stride, int64_t max_pages,
                               void* stream) {
  return rows<true>("sva_paged_write", keys, values, kv_dtype, kv_seq_stride, kv_head_stride, kv_row_stride, n_seq, n_rows,
                    G, D, first_rows, pool, n_pages, page_stride, page_rows, tables, table_stride, max_pages, stream);
}

extern "C" int sva_paged_read(const void* pool, int64_t n_pages, int64_t page_stride, int64_t page_rows,
                              const int32_t* tables, int64_t table_stride, int64_t max_pages, const int64_t* first_rows,
                              int64_t n_seq, int64_t n_rows, int64_t G, int64_t D, void* keys, void* values, int kv_dtype,
                              int64_t kv_seq_stride, int64_t kv_head_stride, int64_t kv_row_stride, void* stream) {
  return rows<false>("sva_paged_read", keys, values, kv_dtype, kv_seq_stride, kv_head_stride, kv_row_stride, n_seq, n_rows,
                     G, D, first_rows, pool, n_pages, page_stride, page_rows, tables, table_stride, max_pages, stream);
}

extern "C" int sva_pages_copy(void* pool, int64_t n_pages, int64_t page_stride_bytes, int64_t layers,
                              int64_t layer_stride_bytes, int64_t page_bytes, const int32_t* src, const int32_t* dst,
                              int64_t n_pairs, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(pool && src && dst, "sva_pages_copy: null pointer");
  SVA_REQUIRE(n_pages > 0 && layers > 0 && page_bytes > 0 && n_pairs > 0 && n_pages < (1ll << 31), "sva_pages_copy: bad sizes");
  SVA_REQUIRE((((uintptr_t)pool | (uintptr_t)page_stride_bytes | (uintptr_t)layer_stride_bytes | (uintptr_t)page_bytes) &
               15u) == 0 && page_stride_bytes >= page_bytes,
              "sva_pages_copy: pages are not blocks of whole aligned 16-byte words");
  SVA_UNSUPPORTED(layers <= 65535, "sva_pages_copy: %lld layers in one call", (long long)layers);
  CopyParams p;
  p.pool = (unsigned char*)pool;
  p.pages = n_pages;
  p.page_bytes = page_stride_bytes;
  p.layer_bytes = layer_stride_bytes;
  p.bytes = page_bytes;
  p.src = src;
  p.dst = dst;
  p.pairs = n_pairs;
  const int64_t pieces = (page_bytes + kPiece - 1) / kPiece;
  SVA_REQUIRE(pieces < (1ll << 31), "sva_pages_copy: pages too large");
  p.pieces = (int)pieces;
  const int64_t y = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(n_pairs, 65535), 16384 / (pieces * layers)));
  hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)pieces, (unsigned)y, (unsigned)layers), dim3(256), 0,
                     (hipStream_t)stream, p);
  SVA_CHECK_LAUNCH("pages_copy_kernel");
  return SVA_OK;
}

extern "C" size_t sva_pages_reserve_workspace_bytes(int64_t n_seq, int64_t n_pages) {
  if (n_seq <= 0 || n_pages <= 0 || reserve_small(n_seq, n_pages)) return 0;
  return (size_t)n_seq * sizeof(Ask) + (size_t)n_pages * sizeof(int32_t);
}

extern "C" int sva_pages_reserve(int32_t* tables, int64_t table_stride, int64_t max_pages, int64_t* seq_lens,
                                 int64_t n_seq, int32_t* refs, int64_t n_pages, int64_t page_rows, const int64_t* counts,
                                 int64_t count, int64_t* first_rows, int32_t* src, int32_t* dst, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(tables && seq_lens && refs && first_rows && src && dst, "sva_pages_reserve: null pointer");
  SVA_REQUIRE(sizes_ok(n_seq, max_pages, n_pages), "sva_pages_reserve: bad sizes");
  SVA_REQUIRE(page_rows_ok(page_rows), "sva_pages_reserve: %lld rows a page are no power of two from 16 to 1024",
              (long long)page_rows);
  const size_t need = sva_pages_reserve_workspace_bytes(n_seq, n_pages);
  SVA_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0 && workspace_bytes >= need),
              "sva_pages_reserve: a workspace of %zu bytes required", need);
  const HoldParams p = hold(tables, table_stride, seq_lens, refs, n_seq, max_pages, n_pages, page_rows);
  Ask* asks = (Ask*)workspace;
  if (need == 0)
    hipLaunchKernelGGL((pages_reserve_kernel<true>), dim3(1), dim3(HB), 0, (hipStream_t)stream, p, counts, count, nullptr,
                       nullptr, first_rows, src, dst);
  else
    hipLaunchKernelGGL((pages_reserve_kernel<false>), dim3(1), dim3(HB), 0, (hipStream_t)stream, p, counts, count, asks,
                       (int32_t*)(asks + n_seq), first_rows, src, dst);
  SVA_CHECK_LAUNCH("pages_reserve_kernel");
  return SVA_OK;
}

extern "C" size_t sva_pages_fork_workspace_bytes(int64_t n_seq, int64_t max_pages) {
  if (n_seq <= 0 || max_pages <= 0 || n_seq * max_pages <= kFewEntries) return 0;
  return (size_t)n_seq * sizeof(int64_t) + (size_t)n_seq * (size_t)max_pages * sizeof(int32_t);
}

extern "C" int sva_pages_fork(int32_t* tables, int64_t table_stride, int64_t max_pages, int64_t* seq_lens, int64_t n_seq,
                              int32_t* refs, int64_t n_pages, int64_t page_rows, const int64_t* sources, void* workspace,
                              size_t workspace_bytes, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(tables && seq_lens && refs && sources, "sva_pages_fork: null pointer");
  SVA_REQUIRE(sizes_ok(n_seq, max_pages, n_pages), "sva_pages_fork: bad sizes");
  SVA_REQUIRE(page_rows_ok(page_rows), "sva_pages_fork: %lld rows a page are no power of two from 16 to 1024",
              (long long)page_rows);
  const size_t need = sva_pages_fork_workspace_bytes(n_seq, max_pages);
  SVA_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0 && workspace_bytes >= need),
              "sva_pages_fork: a workspace of %zu bytes required", need);
  const HoldParams p = hold(tables, table_stride, seq_lens, refs, n_seq, max_pages, n_pages, page_rows);
  if (need == 0) {
    hipLaunchKernelGGL(pages_fork_few_kernel, dim3(1), dim3(HB), 0, (hipStream_t)stream, p, sources);
    SVA_CHECK_LAUNCH("pages_fork_few_kernel");
    return SVA_OK;
  }
  int64_t* next_lens = (int64_t*)workspace;
  int32_t* next = (int32_t*)(next_lens + n_seq);
  const dim3 grid((unsigned)n_seq, (unsigned)((max_pages + 255) / 256));
  hipLaunchKernelGGL(pages_fork_kernel, grid, dim3(256), 0, (hipStream_t)stream, p, sources, next, next_lens);
  SVA_CHECK_LAUNCH("pages_fork_kernel");
  hipLaunchKernelGGL(pages_forked_kernel, grid, dim3(256), 0, (hipStream_t)stream, p, sources, next, next_lens);
  SVA_CHECK_LAUNCH("pages_forked_kernel");
  return SVA_OK;
}

extern "C" size_t sva_pages_compact_workspace_bytes(int64_t n_pages) {
  return n_pages <= 0 ? 0 : (size_t)n_pages * sizeof(int32_t);
}

extern "C" int sva_pages_compact(int32_t* tables, int64_t table_stride, int64_t max_pages, int64_t n_seq, int32_t* refs,
                                 int64_t n_pages, int32_t* src, int32_t* dst, int32_t* used, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(tables && refs && src && dst && used, "sva_pages_compact: null pointer");
  SVA_REQUIRE(sizes_ok(n_seq, max_pages, n_pages), "sva_pages_compact: bad sizes");
  SVA_REQUIRE(workspace && ((uintptr_t)workspace & 3u) == 0 && workspace_bytes >= sva_pages_compact_workspace_bytes(n_pages),
              "sva_pages_compact: a workspace of %zu bytes required", sva_pages_compact_workspace_bytes(n_pages));
  int32_t* to = (int32_t*)workspace;
  hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(HB), 0, (hipStream_t)stream, refs, n_pages, to, src, dst,
                     n_pages / 2, used);
  SVA_CHECK_LAUNCH("pages_compact_kernel");
  hipLaunchKernelGGL(pages_renamed_kernel, dim3((unsigned)n_seq, (unsigned)((max_pages + 255) / 256)), dim3(256), 0,
                     (hipStream_t)stream, tables, table_stride, max_pages, n_pages, to, used);
  SVA_CHECK_LAUNCH("pages_renamed_kernel");
  return SVA_OK;
}
