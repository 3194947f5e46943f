// libosmos MI355X - the paged cache of keys and values (include/osmos_attn.h): rows written into the pages
// (osmos_kv_append) and the pages' own bookkeeping on the device (osmos_kv_grow, _fork, _free, _compact, _copy).
#include "kvcache.h"

namespace osm {
namespace kv {

// ---- append. a wave a row: its lanes take the row's 8-value pieces of k and v in turn, the loads of four in flight while
// the row's sequence and page are looked up (start, len and table are a chain of dependent loads, the rows themselves are
// not). 48 rows of 2 x 8 x 128 floats: 3.7 us, the launch and that chain; 8256 rows of 2 x 4 x 128 bf16 into 8 bits: 9.2 us
// for 25 MB, the same chain in every wave of the one round that the chip holds ----
constexpr int kAppendRows = 4;  // rows (waves) a workgroup

// x / f, each quotient rounded to nearest as a division's, for what is then saturated at 448: by f's reciprocal r, rounded to
// nearest, and q + r (x - f q), exact in its remainder (Markstein's theorem; q may be more than one step off, which it does not
// cover: on the host every mantissa of f with the seven x around each of e4m3's edges and 1.5e9 random pairs gave the division's
// bits). values past 1000 f, infinities among them, are taken as that. three instructions a value where a division is some
// twelve: 8256 rows of 2 x 4 x 128 10.7 -> 10.0 us
__device__ inline void divide8(float (&x)[8], float f) {
  const float size = fabsf(f);
  if (size > 0x1p-60f && size < 0x1p60f) {
    const float r = __fdiv_rn(1.0f, f), most = 1000.0f * size;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float y = __builtin_amdgcn_fmed3f(x[j], -most, most), q = y * r;
      const float z = __builtin_fmaf(__builtin_fmaf(-q, f, y), r, q);
      x[j] = x[j] != x[j] ? x[j] : z;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __fdiv_rn(x[j], f);
  }
}

template <uint32_t SRC, uint32_t DST>
__global__ __launch_bounds__(64 * kAppendRows) void append_kernel(const uint8_t* __restrict__ k, uint64_t ks,
                                                                  const uint8_t* __restrict__ v, uint64_t vs, Step st,
                                                                  uint8_t* __restrict__ data, const float* __restrict__ scale,
                                                                  uint32_t pages, uint32_t page, uint32_t heads, uint32_t dim,
                                                                  uint64_t plane) {
  const uint32_t t = blockIdx.x * kAppendRows + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (t >= st.n_tok) return;
  const uint32_t half = heads * dim / 8, pieces = 2 * half, per = dim / 8;
  float x[4][8];
  auto load = [&](uint32_t c0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t c = c0 + 64 * i;
      if (c >= pieces) break;
      const uint32_t at = c < half ? c : c - half;
      load8<SRC>(c < half ? k + ((uint64_t) t * ks + at * 8ull) * size_of(SRC) : v + ((uint64_t) t * vs + at * 8ull) * size_of(SRC), x[i]);
    }
  };
  load(lane);
  // (every lane takes part in the search, those of a short row that have no piece too)
  Seq q;
  if (!sequence_of(st, (int) t, page, q)) return;
  const int pos = q.len - (q.row0 + q.rows - (int) t);
  if ((int) t < q.row0 || (int) t >= q.row0 + q.rows || pos < 0 || pos >= q.end) return;
  const uint32_t id = (uint32_t) gload<int>(q.table + (uint32_t) pos / page);
  if (id >= pages) return;
  uint8_t* to = data + ((uint64_t) id * heads * page + ((uint32_t) pos & (page - 1))) * dim * size_of(DST);
  for (uint32_t c0 = lane; c0 < pieces;) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t c = c0 + 64 * i;
      if (c >= pieces) break;
      const bool second = c >= half;
      const uint32_t at = second ? c - half : c, h = at / per, d = at - h * per;
      if (DST == OSMOS_F8 && scale) {
        divide8(x[i], scale[(second ? heads : 0) + h]);
      }
      store8<DST>(to + (second ? plane : 0) + ((uint64_t) h * page * dim + d * 8) * size_of(DST), x[i]);
    }
    if ((c0 += 256) < pieces) load(c0);
  }
}

// ---- the pool: one workgroup decides (the outcome goes by the requests' order, and a pool of 65536 pages is 4 rounds of its
// threads' 16 pages each), many copy. a request's pages are the lowest free ids, so a pool that is filled and emptied
// stays near its beginning. growing 24 sequences 7.9 us (a chain of requests, lengths, tables, counts and the list) and 3.6 us for
// 24 copies in 16 planes; compaction of a pool of 4644 pages 8.2 us and 57 us for 278 MB read and written, 4.9 TB/s, what
// a large copy reaches. scratch: list[0 .. pages), then two more such lists (compact's movers and its map), then counts ----

constexpr int kPoolThreads = 1024, kPoolWaves = kPoolThreads / 64, kScan = 16;  // kScan: pages a thread looks over a round

struct Pool {
  int32_t *ref, *len, *table;
  uint32_t pages, page, seqs, width;
};

// exclusive sum of v over the workgroup's threads in their order, *total the whole; `lds`: kPoolWaves + 1 ints
__device__ inline int scan_wg(int v, int* lds, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (the last round's sums have been read)
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPoolWaves; w++) {
    const int s = lds[w];
    before += w < wave ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// the 16 pages from `at` on whose count is zero (free) or not, as bits
__device__ inline uint32_t pages_at(const int32_t* __restrict__ ref, uint32_t at, uint32_t pages, bool free) {
  uint32_t m = 0;
  if (at + kScan <= pages) {
    int4 r[kScan / 4];
#pragma unroll
    for (int i = 0; i < kScan / 4; i++) r[i] = ((const int4*) (ref + at))[i];
#pragma unroll
    for (int i = 0; i < kScan / 4; i++)
      m |= (uint32_t) (r[i].x <= 0) << (4 * i) | (uint32_t) (r[i].y <= 0) << (4 * i + 1) |
           (uint32_t) (r[i].z <= 0) << (4 * i + 2) | (uint32_t) (r[i].w <= 0) << (4 * i + 3);
    return free ? m : ~m & 0xFFFFu;
  }
  for (uint32_t i = 0; i < kScan && at + i < pages; i++) m |= (uint32_t) ((ref[at + i] <= 0) == free) << i;
  return m;
}

// the free (or used) pages of from .. to - 1 in ascending order into list, at most `most`; how many were found
__device__ inline int list_pages(const int32_t* __restrict__ ref, uint32_t from, uint32_t to, bool free, int most,
                                 int32_t* list, int* lds) {
  int found = 0;
  for (uint64_t base = from & ~(uint32_t) (kScan - 1); base < to && found < most; base += (uint64_t) kPoolThreads * kScan) {
    const uint64_t at = base + (uint64_t) threadIdx.x * kScan;
    uint32_t m = at < to ? pages_at(ref, (uint32_t) at, to, free) : 0;
    if (at < from) m &= 0xFFFFu << (from - (uint32_t) at) & 0xFFFFu;
    int all;
    int r = found + scan_wg(__popc(m), lds, &all);
    while (m && r < most) {
      list[r++] = (int32_t) ((uint32_t) at + __builtin_ctz(m));
      m &= m - 1;
    }
    found += all;
  }
  return found < most ? found : most;
}

__global__ __launch_bounds__(kPoolThreads) void grow_kernel(Pool p, const int32_t* __restrict__ seq,
                                                            const int32_t* __restrict__ add, uint32_t n,
                                                            int32_t* __restrict__ list, int2* __restrict__ copies,
                                                            int32_t* __restrict__ done) {
  __shared__ int lds[kPoolWaves + 1], id[OSMOS_KV_MAX_REQUESTS], last[OSMOS_KV_MAX_REQUESTS], have[OSMOS_KV_MAX_REQUESTS],
      first[OSMOS_KV_MAX_REQUESTS + 1], own[OSMOS_KV_MAX_REQUESTS];
  const uint32_t i = threadIdx.x;
  const int s = i < n ? seq[i] : -1;
  id[i] = s;
  __syncthreads();
  bool ok = i < n && (uint32_t) s < p.seqs;
  if (ok)
    for (uint32_t j = 0; j < i; j++) ok = ok && id[j] != s;
  int old = 0, more = 0, held = 0, want = 0, shared = -1;
  if (ok) {
    old = p.len[s], more = add[i];
    const int64_t now = (int64_t) old + more;
    ok = old >= 0 && more >= 0 && now <= 0x7FFFFFFFll && (uint64_t) now <= (uint64_t) p.width * p.page;
    if (ok) {
      held = (int) (((uint32_t) old + p.page - 1) / p.page), want = (int) (((uint32_t) now + p.page - 1) / p.page);
      if (more && (uint32_t) old % p.page) shared = p.table[(uint64_t) s * p.width + held - 1];
      if ((uint32_t) shared >= p.pages) shared = -1;
    }
  }
  last[i] = shared, have[i] = held;
  __syncthreads();
  // a request whose last page has other holders, after the earlier requests took copies of their own, takes one too
  bool cow = false;
  if (shared >= 0) {
    int before = 0;
    for (uint32_t j = 0; j < i; j++) before += last[j] == shared;
    cow = p.ref[shared] - before > 1;
  }
  int total;
  int need = ok ? want - held + cow : 0;
  // (sums past the pages are refused anyway: capped so that they cannot wrap)
  need = need > (int) p.pages ? (int) p.pages + 1 : need;
  int at = 0;
  {  // 64-bit care: n <= 1024 requests of at most 2^31 - 15 pages each could wrap an int sum, so it is taken in units of 2^11
    const int hi = scan_wg(need >> 11, lds, &total);
    const int his = total;
    const int lo = scan_wg(need & 2047, lds, &total);
    const int64_t before = ((int64_t) hi << 11) + lo, all = ((int64_t) his << 11) + total;
    at = before > p.pages ? (int) p.pages + 1 : (int) before;
    total = all > p.pages ? (int) p.pages : (int) all;
  }
  const int free = list_pages(p.ref, 0, p.pages, true, total, list, lds);
  const bool fits = (int64_t) at + need <= free;
  ok = ok && fits;
  first[i] = at;
  if (i == 0) first[kPoolThreads] = 0x7FFFFFFF;
  own[i] = ok ? need : 0;
  __syncthreads();  // (the list and the requests' places in it; every read of ref and table above)
  if (i < n) {
    if (done) done[i] = ok;
    copies[i] = make_int2(ok && cow ? shared : -1, ok && cow ? list[at] : -1);
    if (ok) {
      p.len[s] = old + more;
      if (cow) atomicSub(&p.ref[shared], 1);
    }
    have[i] = held - (cow ? 1 : 0);  // (the first of its pages' place in its table)
  }
  __syncthreads();
  for (int r = (int) i; r < free; r += kPoolThreads) {
    uint32_t a = 0, b = n;  // the last request whose pages start at or before r: the one with pages, as the next starts past r
    while (b - a > 1) {
      const uint32_t m = (a + b) / 2;
      if (first[m] <= r) a = m;
      else b = m;
    }
    if (r - first[a] >= own[a]) continue;  // (pages found for a request that was refused)
    p.table[(uint64_t) id[a] * p.width + have[a] + (r - first[a])] = list[r];
    p.ref[list[r]] = 1;
  }
}

__global__ __launch_bounds__(256) void fork_kernel(Pool p, const int32_t* __restrict__ from, const int32_t* __restrict__ to,
                                                   uint32_t n, int32_t* __restrict__ done) {
  const uint32_t i = blockIdx.x;
  const int a = from[i], b = to[i];
  bool bad = (uint32_t) a >= p.seqs || (uint32_t) b >= p.seqs;
  for (uint32_t j = threadIdx.x; j < n; j += 256) bad = bad || to[j] == a || (j < i && to[j] == b);
  if (!bad) bad = p.len[b] != 0;  // (no other request that is not refused has this `to`)
  bad = __syncthreads_or(bad);
  const int len = bad ? 0 : p.len[a];
  const uint32_t used = len > 0 ? ((uint32_t) len + p.page - 1) / p.page : 0;
  bad = bad || len < 0 || used > p.width;
  if (threadIdx.x == 0 && done) done[i] = !bad;
  if (bad) return;
  for (uint32_t j = threadIdx.x; j < p.width; j += 256) {
    const int page = j < used ? p.table[(uint64_t) a * p.width + j] : -1;
    p.table[(uint64_t) b * p.width + j] = page;
    if ((uint32_t) page < p.pages) atomicAdd(&p.ref[page], 1);
  }
  if (threadIdx.x == 0) p.len[b] = len;  // (read above by this workgroup alone, and before the barrier)
}

__global__ __launch_bounds__(256) void free_kernel(Pool p, const int32_t* __restrict__ seq) {
  __shared__ int mine;
  const int s = seq[blockIdx.x];
  if ((uint32_t) s >= p.seqs) return;
  if (threadIdx.x == 0) mine = atomicExch(&p.len[s], 0);  // (one of the workgroups that name s gets its tokens)
  __syncthreads();
  uint32_t used = mine > 0 ? ((uint32_t) mine + p.page - 1) / p.page : 0;
  if (used > p.width) used = p.width;
  for (uint32_t j = threadIdx.x; j < used; j += 256) {
    int32_t* e = p.table + (uint64_t) s * p.width + j;
    const int page = *e;
    *e = -1;
    if ((uint32_t) page < p.pages) atomicSub(&p.ref[page], 1);
  }
}

// compact's plan: counts[0] = how many pages are in use, counts[1] = how many move, list[j] the j-th free id below that,
// move[j] the j-th used page past it, map[page] its new id; the counts of the pages moved with them
__global__ __launch_bounds__(kPoolThreads) void plan_kernel(Pool p, int32_t* __restrict__ list, int32_t* __restrict__ move,
                                                            int32_t* __restrict__ map, int32_t* __restrict__ counts,
                                                            int32_t* __restrict__ live) {
  __shared__ int lds[kPoolWaves + 1];
  int used = 0;
  for (uint64_t at = (uint64_t) threadIdx.x * kScan; at < p.pages; at += (uint64_t) kPoolThreads * kScan)
    used += __popc(pages_at(p.ref, (uint32_t) at, p.pages, false));
  int n;
  scan_wg(used, lds, &n);
  const int moved = list_pages(p.ref, 0, (uint32_t) n, true, n, list, lds);
  list_pages(p.ref, (uint32_t) n, p.pages, false, moved, move, lds);
  __syncthreads();
  for (int j = (int) threadIdx.x; j < moved; j += kPoolThreads) {
    const int a = move[j], b = list[j];
    map[a] = b;
    p.ref[b] = p.ref[a];
    p.ref[a] = 0;
  }
  if (threadIdx.x == 0) {
    counts[0] = n, counts[1] = moved;
    if (live) *live = n;
  }
}

// the bytes of one page of one plane, a part a workgroup: 16 bytes a thread, four in flight
constexpr uint32_t kPart = 256 * 16 * 4;

__device__ inline void copy_part(uint8_t* __restrict__ data, uint64_t bytes, uint64_t plane, uint32_t pl, uint32_t part,
                                 uint32_t a, uint32_t b) {
  const uint8_t* from = data + pl * plane + a * bytes;
  uint8_t* to = data + pl * plane + b * bytes;
  const uint64_t at = (uint64_t) part * kPart + threadIdx.x * 16;
  u32x4 w[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (at + i * 4096 < bytes) w[i] = gload<u32x4>(from + at + i * 4096);
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (at + i * 4096 < bytes) *(u32x4*) (to + at + i * 4096) = w[i];
}

// page pairs, from[i * step] and to[i * step]: a workgroup takes parts of them in turn
__global__ __launch_bounds__(256) void copy_kernel(uint8_t* data, uint64_t bytes, uint64_t plane, uint32_t planes,
                                                   uint32_t parts, uint32_t pages, const int32_t* __restrict__ from,
                                                   const int32_t* __restrict__ to, uint32_t step, uint32_t n) {
  const uint64_t each = (uint64_t) planes * parts, all = each * n;
  for (uint64_t u = blockIdx.x; u < all; u += gridDim.x) {
    const uint32_t i = (uint32_t) (u / each), rest = (uint32_t) (u - i * each), pl = rest / parts;
    const uint32_t a = (uint32_t) from[(uint64_t) i * step], b = (uint32_t) to[(uint64_t) i * step];
    if (a < pages && b < pages) copy_part(data, bytes, plane, pl, rest - pl * parts, a, b);
  }
}

// compact's moves, and the tables' ids after them
__global__ __launch_bounds__(256) void move_kernel(Pool p, uint8_t* data, uint64_t bytes, uint64_t plane, uint32_t planes,
                                                   uint32_t parts, const int32_t* __restrict__ list,
                                                   const int32_t* __restrict__ move, const int32_t* __restrict__ map,
                                                   const int32_t* __restrict__ counts) {
  const uint32_t n = (uint32_t) counts[0], moved = (uint32_t) counts[1];
  if (!moved) return;
  const uint64_t entries = (uint64_t) p.seqs * p.width;
  for (uint64_t e = (uint64_t) blockIdx.x * 256 + threadIdx.x; e < entries; e += (uint64_t) gridDim.x * 256) {
    const uint32_t s = (uint32_t) (e / p.width), j = (uint32_t) (e - (uint64_t) s * p.width);
    const int len = p.len[s];
    const uint32_t page = (uint32_t) p.table[e];
    if (len > 0 && j < ((uint32_t) len + p.page - 1) / p.page && page >= n && page < p.pages) p.table[e] = map[page];
  }
  const uint64_t each = (uint64_t) planes * parts, all = each * moved;
  for (uint64_t u = blockIdx.x; u < all; u += gridDim.x) {
    const uint32_t i = (uint32_t) (u / each), rest = (uint32_t) (u - i * each), pl = rest / parts;
    copy_part(data, bytes, plane, pl, rest - pl * parts, (uint32_t) move[i], (uint32_t) list[i]);
  }
}

constexpr uint32_t kCopyGrid = 4096;

inline uint32_t parts_of(const OsmosKv* kv) { return (uint32_t) ((page_bytes(kv) + kPart - 1) / kPart); }
inline uint32_t copy_grid(const OsmosKv* kv, uint64_t pairs) {
  const uint64_t n = pairs * 2 * kv->layers * parts_of(kv);
  return (uint32_t) (n < kCopyGrid ? n : kCopyGrid);
}
inline Pool pool_of(const OsmosKv* kv, const OsmosKvPool* p) {
  return Pool{p->ref, p->len, p->table, kv->pages, kv->page, p->seqs, p->table_stride};
}

template <uint32_t SRC>
inline auto append_to(uint32_t type) {
  return type == OSMOS_F16 ? append_kernel<SRC, OSMOS_F16> : type == OSMOS_BF16 ? append_kernel<SRC, OSMOS_BF16> : append_kernel<SRC, OSMOS_F8>;
}

}  // namespace kv
}  // namespace osm

using namespace osm;

extern "C" OSM_API uint64_t osmos_kv_bytes(const OsmosKv* kv) {
  return kv::shape_ok(kv) ? 2ull * kv->layers * kv::plane_bytes(kv) : 0;
}

extern "C" OSM_API bool osmos_kv_append(const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step, uint32_t type,
                                        const void* k, uint64_t k_stride, const void* v, uint64_t v_stride, void* stream) {
  if (!kv::append_ok(kv, layer, step, type, k, k_stride, v, v_stride)) return false;
  const uint64_t plane = kv::plane_bytes(kv);
  auto* kernel = type == OSMOS_F32 ? kv::append_to<OSMOS_F32>(kv->type) : type == OSMOS_F16 ? kv::append_to<OSMOS_F16>(kv->type) : kv::append_to<OSMOS_BF16>(kv->type);
  kernel<<<(step->n_tok + kv::kAppendRows - 1) / kv::kAppendRows, 64 * kv::kAppendRows, 0, (hipStream_t) stream>>>(
      (const uint8_t*) k, k_stride, (const uint8_t*) v, v_stride, kv::step_of(step), (uint8_t*) kv->data + 2ull * layer * plane,
      kv->scale ? kv->scale + 2ull * layer * kv->heads : nullptr, kv->pages, kv->page, kv->heads, kv->dim, plane);
  return hipGetLastError() == hipSuccess;
}

extern "C" OSM_API uint64_t osmos_kv_scratch(const OsmosKv* kv) {
  return kv::shape_ok(kv) ? (3 * kv::list_ints(kv) + 2 * OSMOS_KV_MAX_REQUESTS + 16) * 4 : 0;
}

extern "C" OSM_API bool osmos_kv_grow(const OsmosKv* kv, const OsmosKvPool* pool, const int32_t* seq, const int32_t* add,
                                      uint32_t n, int32_t* done, void* stream) {
  if (!kv::requests_ok(kv, pool, seq, add, n)) return false;
  int32_t* list = (int32_t*) pool->scratch;
  int2* copies = (int2*) (list + 3 * kv::list_ints(kv));
  kv::grow_kernel<<<1, kv::kPoolThreads, 0, (hipStream_t) stream>>>(kv::pool_of(kv, pool), seq, add, n, list, copies, done);
  if (hipGetLastError() != hipSuccess) return false;
  kv::copy_kernel<<<kv::copy_grid(kv, n), 256, 0, (hipStream_t) stream>>>(
      (uint8_t*) kv->data, kv::page_bytes(kv), kv::plane_bytes(kv), 2 * kv->layers, kv::parts_of(kv), kv->pages,
      (const int32_t*) copies, (const int32_t*) copies + 1, 2, n);
  return hipGetLastError() == hipSuccess;
}

extern "C" OSM_API bool osmos_kv_fork(const OsmosKv* kv, const OsmosKvPool* pool, const int32_t* from, const int32_t* to,
                                      uint32_t n, int32_t* done, void* stream) {
  if (!kv::requests_ok(kv, pool, from, to, n)) return false;
  kv::fork_kernel<<<n, 256, 0, (hipStream_t) stream>>>(kv::pool_of(kv, pool), from, to, n, done);
  return hipGetLastError() == hipSuccess;
}

extern "C" OSM_API bool osmos_kv_free(const OsmosKv* kv, const OsmosKvPool* pool, const int32_t* seq, uint32_t n,
                                      void* stream) {
  if (!kv::requests_ok(kv, pool, seq, seq, n)) return false;
  kv::free_kernel<<<n, 256, 0, (hipStream_t) stream>>>(kv::pool_of(kv, pool), seq);
  return hipGetLastError() == hipSuccess;
}

extern "C" OSM_API bool osmos_kv_compact(const OsmosKv* kv, const OsmosKvPool* pool, int32_t* live, void* stream) {
  if (!kv::pool_ok(kv, pool)) return false;
  const uint64_t ints = kv::list_ints(kv);
  int32_t *list = (int32_t*) pool->scratch, *move = list + ints, *map = move + ints, *counts = map + ints;
  kv::plan_kernel<<<1, kv::kPoolThreads, 0, (hipStream_t) stream>>>(kv::pool_of(kv, pool), list, move, map, counts, live);
  if (hipGetLastError() != hipSuccess) return false;
  kv::move_kernel<<<kv::copy_grid(kv, kv->pages), 256, 0, (hipStream_t) stream>>>(
      kv::pool_of(kv, pool), (uint8_t*) kv->data, kv::page_bytes(kv), kv::plane_bytes(kv), 2 * kv->layers, kv::parts_of(kv),
      list, move, map, counts);
  return hipGetLastError() == hipSuccess;
}

extern "C" OSM_API bool osmos_kv_copy(const OsmosKv* kv, const int32_t* from, const int32_t* to, uint32_t n, void* stream) {
  if (!kv::copy_ok(kv, from, to, n)) return false;
  kv::copy_kernel<<<kv::copy_grid(kv, n), 256, 0, (hipStream_t) stream>>>(
      (uint8_t*) kv->data, kv::page_bytes(kv), kv::plane_bytes(kv), 2 * kv->layers, kv::parts_of(kv), kv->pages, from, to, 1, n);
  return hipGetLastError() == hipSuccess;
}
