// Pages of the paged K/V cache: reserve (with copy on write), fork, truncate,
// copy, compact, append; and the C ABI of the cache (include/moe_sm100.h).
//
// State, all in the caller's device memory: block_table[seq][block] (page or -1),
// lengths[seq], refs[page] (sequences that hold it, 0 = free).  A page is free when
// no sequence holds it, so freeing is a decrement and needs no free list: two
// sequences that let go of a page in one call give the same state in either order.
// A call that allocates takes the lowest free pages in the order of its entries, so
// the tables do not depend on the order in which blocks or atomics run.
//
// A call checks its sequence indices (range, the same one twice) before it changes
// anything and refuses as a whole; an entry whose own state forbids the step (a
// child that is not empty, a longer new length) is left as it was.  A batch of rows is
// refused as a whole for its offsets and for a sequence with rows in two entries; an entry
// without a sequence and a row without a place are left out.  All are reported by
// moe_kv_status.
#include <algorithm>
#include <new>
#include <string>

#include "common.cuh"
#include "kv_internal.h"

namespace moe {

constexpr int kPlanThreads = 1024;  // the one-CTA planning kernels

// Inclusive sum over the CTA (blockDim.x = 32 * NW); *total gets the whole sum.
template <int NW>
MOE_DEV unsigned long long block_scan(unsigned long long v, unsigned long long* total) {
  __shared__ unsigned long long part[NW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    unsigned long long p = lane < NW ? part[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += u;
    }
    if (lane < NW) part[lane] = p;
  }
  __syncthreads();
  *total = part[NW - 1];
  const unsigned long long before = warp ? part[warp - 1] : 0;
  __syncthreads();  // part is written again by the next call
  return v + before;
}

// True for every thread when each of seqs[0..n) is a sequence and none comes twice;
// bits: nseq bits of shared memory.
MOE_DEV bool seqs_ok(const int* __restrict__ seqs, int n, int nseq, uint32_t* bits) {
  for (int i = threadIdx.x; i < (nseq + 31) / 32; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = seqs[i];
    if (s < 0 || s >= nseq) {
      bad = true;
    } else if (atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) {
      bad = true;
    }
  }
  return !__syncthreads_or(bad);
}

MOE_DEV int blocks_of(const KvView& c, int tokens) {
  return static_cast<int>((static_cast<int64_t>(tokens) + c.page - 1) >> c.page_shift);
}

// ------------------------------------------------------------------ reserve
// One CTA: (1) the pages that each entry needs (a fresh copy of a shared, partly
// filled last page among them) and their prefix sum, (2) the lowest free pages, as
// many as needed, (3) hand them out in entry order.  Nothing is written to the
// cache before the whole call is known to succeed.
__global__ void __launch_bounds__(kPlanThreads) kv_reserve_kernel(const KvView c,
                                                                  const int* __restrict__ seqs,
                                                                  const int* __restrict__ counts,
                                                                  int n) {
  pdl_enter();
  extern __shared__ uint32_t bits[];
  const int tid = threadIdx.x;
  if (tid == 0) *c.count = 0;
  if (!seqs_ok(seqs, n, c.nseq, bits)) {
    if (tid == 0) record_error(c.err, DEV_BAD_SEQ);
    return;
  }
  // (1) low 44 bits: pages needed before entry i; high 20: copies before it
  constexpr int kCopyBit = 44;
  unsigned long long run = 0;
  bool bad = false;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    unsigned long long need = 0;
    if (i < n) {
      const int s = seqs[i], have = c.len[s], more = counts[i];
      const int64_t after = static_cast<int64_t>(have) + more;
      if (have < 0 || more < 0 || after > static_cast<int64_t>(c.max_blocks) << c.page_shift ||
          after > 0x7fffffff) {
        bad = true;
      } else {
        const int nb = blocks_of(c, have);
        // more than the pool holds fails whatever the number: capped, the sums fit
        need = min(blocks_of(c, static_cast<int>(after)) - nb, c.pages + 1);
        if (more > 0 && (have & (c.page - 1))) {
          const int pg = c.table[static_cast<int64_t>(s) * c.max_blocks + nb - 1];
          if (pg < 0 || pg >= c.pages) bad = true;
          else if (c.refs[pg] > 1) need += 1 | (1ull << kCopyBit);
        }
      }
    }
    unsigned long long total;
    const unsigned long long incl = run + block_scan<32>(need, &total);
    if (i < n) c.off[i] = static_cast<int>(incl - need);  // low word: pages
    // an entry's copy goes to slot (copies before it); kept beside it for step (3)
    if (i < n) c.rows[i] = (need >> kCopyBit) ? static_cast<int>((incl >> kCopyBit) - 1) : -1;
    run += total;
  }
  const unsigned long long wanted = run & ((1ull << kCopyBit) - 1);
  const int want = static_cast<int>(min(wanted, static_cast<unsigned long long>(c.pages) + 1));
  if (__syncthreads_or(bad)) {
    if (tid == 0) record_error(c.err, DEV_BAD_LENGTH);
    return;
  }
  // (2) sixteen pages a thread and step
  int found = 0;
  for (int64_t p0 = 0; p0 < c.pages && found < want; p0 += 16 * kPlanThreads) {
    const int64_t p = p0 + 16 * tid;
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (p + j < c.pages && c.refs[p + j] == 0) mask |= 1u << j;
    unsigned long long total;
    int at = found + static_cast<int>(block_scan<32>(__popc(mask), &total)) - __popc(mask);
    for (; mask && at < want; mask &= mask - 1) c.list[at++] = static_cast<int>(p) + __ffs(mask) - 1;
    found += static_cast<int>(total);
  }
  if (found < want) {
    if (tid == 0) record_error(c.err, DEV_NO_PAGES);
    return;
  }
  __syncthreads();
  // (3) a thread per entry; entries with many pages by their whole warp.  A copy's slot is
  // its rank among the copies, at most its entry's number: rows[] of a chunk is read by all
  // threads before any slot of it is written.
  const int lane = tid & 31;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int s = 0, have = 0, more = 0, slot = -1, from = 0;
    if (i < n) {
      s = seqs[i];
      more = counts[i];
      slot = c.rows[i];
      from = c.off[i];
      have = c.len[s];
    }
    int* row = c.table + static_cast<int64_t>(s) * c.max_blocks;
    const int first = blocks_of(c, have), last = more > 0 ? blocks_of(c, have + more) : first;
    __syncthreads();
    if (slot >= 0) {
      const int old = row[first - 1], fresh = c.list[from++];
      row[first - 1] = fresh;
      c.refs[fresh] = 1;
      atomicSub(&c.refs[old], 1);
      c.src[slot] = old;
      c.dst[slot] = fresh;
      c.rows[slot] = have & (c.page - 1);
    }
    const bool many = last - first > 4;
    if (!many) {
      for (int j = first; j < last; ++j) {
        const int pg = c.list[from + j - first];
        row[j] = pg;
        c.refs[pg] = 1;
      }
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, many); todo; todo &= todo - 1) {
      const int l = __ffs(todo) - 1;
      const int at = __shfl_sync(0xffffffffu, first, l), to = __shfl_sync(0xffffffffu, last, l);
      const int lf = __shfl_sync(0xffffffffu, from, l), ls = __shfl_sync(0xffffffffu, s, l);
      for (int j = at + lane; j < to; j += 32) {
        const int pg = c.list[lf + j - at];
        c.table[static_cast<int64_t>(ls) * c.max_blocks + j] = pg;
        c.refs[pg] = 1;
      }
    }
    if (i < n) c.len[s] = have + more;
    __syncthreads();
  }
  if (tid == 0) *c.count = static_cast<int>(run >> kCopyBit);
}

// ------------------------------------------------------------------ page copies
// *count pages src[i] -> dst[i], rows[i] rows of each head (rows null: whole pages),
// every layer, keys and values.  A warp copies the rows of one (page, layer, K or V,
// head), 16 bytes a lane, eight loads in flight: bound by HBM (each byte read and
// written once).  from / to: two pools of the same shape but for their pages, or one.
__global__ void __launch_bounds__(256) kv_copy_kernel(const KvView from, const KvView to,
                                                      const int* __restrict__ rows) {
  pdl_enter();
  const int n = *from.count;
  const int lane = threadIdx.x & 31;
  const int per_page = from.layers * 2 * from.heads;
  const int chunks_shift = from.hd == 128 ? 4 : 3;  // 16-byte chunks of a row
  const int64_t items = static_cast<int64_t>(n) * per_page;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       it < items; it += stride) {
    const int i = static_cast<int>(it / per_page);
    int r = static_cast<int>(it - static_cast<int64_t>(i) * per_page);
    const int h = r % from.heads;
    r /= from.heads;
    const bool val = r & 1;
    const int l = r >> 1;
    const int64_t(&fs)[4] = val ? from.vs : from.ks;
    const int64_t(&ts)[4] = val ? to.vs : to.ks;
    const char* a = (val ? from.v : from.k) + l * fs[0] + from.src[i] * fs[1] + h * fs[2];
    char* b = (val ? to.v : to.k) + l * ts[0] + from.dst[i] * ts[1] + h * ts[2];
    const int nc = (rows ? rows[i] : from.page) << chunks_shift;
    const int cmask = (1 << chunks_shift) - 1;
    // lane's chunk of row r0, and the rows that 32 lanes cover in a step
    const int step = 32 >> chunks_shift;
    const int64_t fstep = step * fs[3], tstep = step * ts[3];
    const char* pa = a + (lane >> chunks_shift) * fs[3] + (lane & cmask) * 16;
    char* pb = b + (lane >> chunks_shift) * ts[3] + (lane & cmask) * 16;
    for (int c0 = lane; c0 < nc; c0 += 256) {
      uint4 q[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c0 + 32 * u < nc) q[u] = *reinterpret_cast<const uint4*>(pa + u * fstep);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c0 + 32 * u < nc) *reinterpret_cast<uint4*>(pb + u * tstep) = q[u];
      pa += 8 * fstep;
      pb += 8 * tstep;
    }
  }
}

// One CTA: checks src / dst of a raw copy (range; a destination that comes twice or
// is also a source would make the result depend on the order) and sets the list.
__global__ void __launch_bounds__(kPlanThreads) kv_copy_plan_kernel(const KvView c,
                                                                    const int* __restrict__ src,
                                                                    const int* __restrict__ dst,
                                                                    int n) {
  pdl_enter();
  const int tid = threadIdx.x;
  if (tid == 0) *c.count = 0;
  bool bad = false;
  for (int i = tid; i < n; i += kPlanThreads) {
    const int a = src[i], b = dst[i];
    bad |= a < 0 || a >= c.pages || b < 0 || b >= c.pages;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) record_error(c.err, DEV_BAD_PAGE);
    return;
  }
  for (int i = tid; i < n; i += kPlanThreads) {
    c.list[src[i]] = 0;
    c.list[dst[i]] = 0;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) bad |= atomicAdd(&c.list[dst[i]], 1) != 0;
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) bad |= c.list[src[i]] != 0;
  if (__syncthreads_or(bad)) {
    if (tid == 0) record_error(c.err, DEV_BAD_PAGE);
    return;
  }
  for (int i = tid; i < n; i += kPlanThreads) {
    c.src[i] = src[i];
    c.dst[i] = dst[i];
  }
  if (tid == 0) *c.count = n;
}

// ------------------------------------------------------------------ fork
// A CTA per pair: the child's table row becomes the parent's, one more reference on
// each page.  Every CTA checks the whole list (a few kilobytes from L2), so that no
// second launch is needed: the indices alone decide, and no CTA changes them.
__global__ void __launch_bounds__(256) kv_fork_kernel(const KvView c,
                                                      const int* __restrict__ parents,
                                                      const int* __restrict__ children, int n) {
  pdl_enter();
  extern __shared__ uint32_t bits[];
  bool ok = seqs_ok(children, n, c.nseq, bits);
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int p = parents[i];
    bad |= p < 0 || p >= c.nseq || (bits[p >> 5] >> (p & 31) & 1u);  // a parent is no child
  }
  if (__syncthreads_or(bad) || !ok) {
    if (threadIdx.x == 0) record_error(c.err, DEV_BAD_SEQ);
    return;
  }
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int p = parents[i], ch = children[i];
    const int len = c.len[p];
    const bool empty = c.len[ch] == 0;
    __syncthreads();  // every thread has read the child's length
    const int nb = blocks_of(c, max(len, 0));
    if (!empty || nb > c.max_blocks) {
      if (threadIdx.x == 0) record_error(c.err, DEV_BAD_LENGTH);
      continue;
    }
    const int* from = c.table + static_cast<int64_t>(p) * c.max_blocks;
    int* to = c.table + static_cast<int64_t>(ch) * c.max_blocks;
    for (int j = threadIdx.x; j < nb; j += blockDim.x) {
      const int pg = from[j];
      to[j] = pg;
      if (pg >= 0 && pg < c.pages) atomicAdd(&c.refs[pg], 1);
      else record_error(c.err, DEV_BAD_PAGE);
    }
    if (threadIdx.x == 0) c.len[ch] = len;
  }
}

// ------------------------------------------------------------------ truncate
// A CTA per entry: the pages past ceil(length / page) lose a reference.
__global__ void __launch_bounds__(256) kv_truncate_kernel(const KvView c,
                                                          const int* __restrict__ seqs,
                                                          const int* __restrict__ lengths, int n) {
  pdl_enter();
  extern __shared__ uint32_t bits[];
  if (!seqs_ok(seqs, n, c.nseq, bits)) {
    if (threadIdx.x == 0) record_error(c.err, DEV_BAD_SEQ);
    return;
  }
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int s = seqs[i], to = lengths[i], have = c.len[s];
    __syncthreads();  // every thread has read the old length
    const int nb = blocks_of(c, max(have, 0));
    if (to < 0 || to > have || nb > c.max_blocks) {
      if (threadIdx.x == 0) record_error(c.err, DEV_BAD_LENGTH);
      continue;
    }
    int* row = c.table + static_cast<int64_t>(s) * c.max_blocks;
    for (int j = blocks_of(c, to) + threadIdx.x; j < nb; j += blockDim.x) {
      const int pg = row[j];
      row[j] = -1;
      if (pg >= 0 && pg < c.pages) atomicSub(&c.refs[pg], 1);
      else record_error(c.err, DEV_BAD_PAGE);
    }
    if (threadIdx.x == 0) c.len[s] = to;
  }
}

// ------------------------------------------------------------------ compact
// One CTA.  Into another pool: the live page of rank r becomes page r.  In place
// (to_pages = 0): live pages already below L, their number, stay; the others fill the
// holes below L, lowest into lowest.  list[page] becomes the new page, src / dst the
// copies, count their number.
__global__ void __launch_bounds__(kPlanThreads) kv_compact_plan_kernel(const KvView c, int to_pages) {
  pdl_enter();
  const int tid = threadIdx.x;
  const bool in_place = to_pages == 0;
  if (tid == 0) *c.count = 0;
  int live = 0;
  if (in_place) {
    unsigned long long mine = 0, total;
    for (int p = tid; p < c.pages; p += kPlanThreads) mine += c.refs[p] > 0;
    block_scan<32>(mine, &total);
    live = static_cast<int>(total);
  }
  int rank = 0, holes = 0, movers = 0;  // so far
  for (int64_t p0 = 0; p0 < c.pages; p0 += 16 * kPlanThreads) {
    const int p = static_cast<int>(p0) + 16 * tid;
    uint32_t used = 0, there = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (p + j < c.pages) {
        there |= 1u << j;
        if (c.refs[p + j] > 0) used |= 1u << j;
      }
    }
    unsigned long long total;
    if (!in_place) {
      int at = rank + static_cast<int>(block_scan<32>(__popc(used), &total)) - __popc(used);
      for (uint32_t m = used; m; m &= m - 1, ++at) {
        const int pg = p + __ffs(m) - 1;
        c.list[pg] = at;
        c.src[at] = pg;
        c.dst[at] = at;
      }
      rank += static_cast<int>(total);
    } else {
      const int below = min(max(live - p, 0), 16);  // pages of these 16 that lie below L
      const uint32_t low = below >= 16 ? 0xffffu : (1u << below) - 1u;
      const uint32_t hole = there & low & ~used, move = used & ~low;
      const unsigned long long both = __popc(hole) | (static_cast<unsigned long long>(__popc(move)) << 32);
      const unsigned long long incl = block_scan<32>(both, &total);
      int hi = holes + static_cast<int>((incl - both) & 0xffffffffu);
      int mv = movers + static_cast<int>((incl - both) >> 32);
      for (uint32_t m = used & low; m; m &= m - 1) c.list[p + __ffs(m) - 1] = p + __ffs(m) - 1;
      // a page that nobody holds goes nowhere, should a table name it
      for (uint32_t m = there & ~used; m; m &= m - 1) c.list[p + __ffs(m) - 1] = -1;
      for (uint32_t m = hole; m; m &= m - 1) c.dst[hi++] = p + __ffs(m) - 1;
      for (uint32_t m = move; m; m &= m - 1) c.src[mv++] = p + __ffs(m) - 1;
      holes += static_cast<int>(total & 0xffffffffu);
      movers += static_cast<int>(total >> 32);
    }
  }
  if (in_place) {
    __syncthreads();
    for (int i = tid; i < movers; i += kPlanThreads) c.list[c.src[i]] = c.dst[i];
    if (tid == 0) *c.count = movers;  // holes == movers: the live pages above L
  } else if (rank > to_pages) {
    if (tid == 0) {
      *c.count = -1;  // the tables stay as they are
      record_error(c.err, DEV_NO_PAGES);
    }
  } else if (tid == 0) {
    *c.count = rank;
  }
}

// Tables, lengths and references after a compaction (to: this cache or another).
__global__ void __launch_bounds__(256) kv_compact_tables_kernel(const KvView c, const KvView to,
                                                                int in_place) {
  pdl_enter();
  const int n = *c.count;
  if (n < 0) return;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t cells = static_cast<int64_t>(to.nseq) * to.max_blocks;
  if (in_place) {
    for (int64_t i = first; i < cells; i += stride) {
      const int pg = c.table[i];
      if (pg >= 0 && pg < c.pages) c.table[i] = c.list[pg];
    }
    for (int64_t i = first; i < n; i += stride) {
      c.refs[c.dst[i]] = c.refs[c.src[i]];
      c.refs[c.src[i]] = 0;
    }
    return;
  }
  for (int64_t i = first; i < cells; i += stride) {
    const int s = static_cast<int>(i / to.max_blocks), b = static_cast<int>(i - static_cast<int64_t>(s) * to.max_blocks);
    int pg = s < c.nseq && b < c.max_blocks ? c.table[static_cast<int64_t>(s) * c.max_blocks + b] : -1;
    // a page that a table names but nobody holds has no place in the other pool
    if (pg >= 0) pg = pg < c.pages && c.refs[pg] > 0 ? c.list[pg] : -1;
    to.table[i] = pg;
  }
  for (int64_t i = first; i < to.nseq; i += stride) to.len[i] = i < c.nseq ? c.len[i] : 0;
  for (int64_t i = first; i < to.pages; i += stride) to.refs[i] = i < n ? c.refs[c.src[i]] : 0;
}

// ------------------------------------------------------------------ append
// A warp per row: all heads of the row's key, then of its value, 16 bytes a lane.
// Bound by HBM for long chunks (each byte read and written once; 10,168 rows of 8 heads, 83
// MB: 16.6 us, 5.0 TB/s), by the launch and three dependent loads (entry, length, page) for
// a decode step (64 rows: 3.0 us, 0.3 of them the check of the batch).
__global__ void __launch_bounds__(128, 8) kv_append_kernel(const KvView c, const KvBatch b, int layer,
                                                        const char* __restrict__ k,
                                                        const char* __restrict__ v, int64_t kt,
                                                        int64_t kh, int64_t vt, int64_t vh) {
  pdl_enter();
  extern __shared__ uint32_t bits[];
  if (!batch_ok(c, b, bits)) return;
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5);
  const int total = b.q_start[b.n];
  const int shift = c.hd == 128 ? 4 : 3;  // chunks of a head
  const int nc = c.heads << shift;
  for (int r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < total; r += warps) {
    const int e = entry_of_row(b.q_start, b.n, r);
    if (e < 0) continue;  // q_start[0] > r: no entry's row
    const int s = b.seqs[e];
    if (s < 0 || s >= c.nseq) {
      if (lane == 0) record_error(c.err, DEV_BAD_SEQ);
      continue;
    }
    const int64_t pos = static_cast<int64_t>(c.len[s]) - (b.q_start[e + 1] - r);
    const int64_t blk = pos >> c.page_shift;
    const int pg = pos >= 0 && blk < c.max_blocks ? c.table[static_cast<int64_t>(s) * c.max_blocks + blk] : -1;
    if (pg < 0 || pg >= c.pages) {
      if (lane == 0) record_error(c.err, pos < 0 ? DEV_BAD_LENGTH : DEV_BAD_PAGE);
      continue;
    }
    const int64_t slot = pos & (c.page - 1);
    char* dk = c.k + layer * c.ks[0] + pg * c.ks[1] + slot * c.ks[3];
    char* dv = c.v + layer * c.vs[0] + pg * c.vs[1] + slot * c.vs[3];
    const char* sk = k + r * kt;
    const char* sv = v + r * vt;
    for (int c0 = lane; c0 < nc; c0 += 128) {
      uint4 qk[4], qv[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int ch = c0 + 32 * u, h = ch >> shift, o = (ch & ((1 << shift) - 1)) * 16;
        if (ch < nc) {
          qk[u] = *reinterpret_cast<const uint4*>(sk + h * kh + o);
          qv[u] = *reinterpret_cast<const uint4*>(sv + h * vh + o);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int ch = c0 + 32 * u, h = ch >> shift, o = (ch & ((1 << shift) - 1)) * 16;
        if (ch < nc) {
          *reinterpret_cast<uint4*>(dk + h * c.ks[2] + o) = qk[u];
          *reinterpret_cast<uint4*>(dv + h * c.vs[2] + o) = qv[u];
        }
      }
    }
  }
}

// One CTA: the check of a batch of more than kCheckHere entries.
__global__ void __launch_bounds__(kPlanThreads) kv_check_kernel(const KvView c, const KvBatch b) {
  pdl_enter();
  extern __shared__ uint32_t bits[];
  const bool ok = check_batch<4>(c, b, bits);
  if (threadIdx.x == 0) *c.ok = ok;
}
cudaError_t kv_launch_check(const KvView& c, const KvBatch& b, cudaStream_t s) {
  if (b.n <= kCheckHere) return cudaSuccess;
  return pdl_launch(kv_check_kernel, dim3(1), dim3(kPlanThreads), bitmap_bytes(c), s, c, b);
}

cudaError_t kv_launch_append(const KvView& c, const KvBatch& b, int layer, const void* k,
                             const void* v, const int64_t (&ks)[2], const int64_t (&vs)[2],
                             int num_sms, cudaStream_t s) {
  const int grid = std::min((b.rows + 3) / 4, num_sms * 16);
  const cudaError_t st = kv_launch_check(c, b, s);
  if (st != cudaSuccess) return st;
  return pdl_launch(kv_append_kernel, dim3(grid), dim3(128), bitmap_bytes(c), s, c, b, layer,
                    static_cast<const char*>(k), static_cast<const char*>(v), ks[0] * 2, ks[1] * 2,
                    vs[0] * 2, vs[1] * 2);
}

}  // namespace moe

// ====================================================================== C ABI
using namespace moe;

namespace {

int kfail(int code, const char* msg) {
  set_error(msg);
  return code;
}
int kfail(int code, const std::string& msg) { return kfail(code, msg.c_str()); }

// The cache's device is current inside a call and the caller's again after it.
struct DeviceScope {
  int before = -1;
  cudaError_t st;
  explicit DeviceScope(int device) {
    st = cudaGetDevice(&before);
    if (st == cudaSuccess && before != device) {
      st = cudaSetDevice(device);
    } else {
      before = -1;
    }
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

#define MOE_KV_ENTER(cache)                                                            \
  if (!(cache)) return kfail(MOE_ERR_INVALID, "null cache");                           \
  DeviceScope scope((cache)->device);                                                  \
  if (scope.st != cudaSuccess)                                                         \
    return kfail(MOE_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(scope.st))

#define MOE_KV_CUDA(call)                                                              \
  do {                                                                                 \
    const cudaError_t st_ = (call);                                                    \
    if (st_ != cudaSuccess)                                                            \
      return kfail(MOE_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(st_)); \
  } while (0)

// enough CTAs to fill the GPU for any number of pages (the count is on the device)
dim3 copy_grid(const MoeKvCache* c) { return dim3(c->num_sms * 8); }

bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }

int check_batch(const MoeKvCache* c, int32_t layer, const int32_t* seqs, const int32_t* q_start,
                int32_t n, int32_t rows) {
  if (n < 0 || rows < 0) return kfail(MOE_ERR_INVALID, "negative n_seqs or rows");
  if (layer < 0 || layer >= c->v.layers) return kfail(MOE_ERR_INVALID, "layer outside the cache");
  if (n > 0 && rows > 0 && (!seqs || !q_start)) return kfail(MOE_ERR_INVALID, "null seqs / q_start");
  return MOE_OK;
}

bool bad_strides(const int64_t* s) { return s[0] < 0 || s[1] < 0 || s[0] % 8 || s[1] % 8; }

}  // namespace

extern "C" {

uint64_t moe_kv_scratch_bytes(const MoeKvConfig* cfg) {
  if (!cfg || cfg->pages <= 0 || cfg->sequences <= 0) return 0;
  return kv_scratch_words(cfg->pages, cfg->sequences) * 4;
}

int moe_kv_create(const MoeKvConfig* cfg, MoeKvCache** out) {
  if (!cfg || !out) return kfail(MOE_ERR_INVALID, "null argument");
  const MoeKvConfig& c = *cfg;
  if (c.dtype != MOE_KV_F16 && c.dtype != MOE_KV_BF16)
    return kfail(MOE_ERR_UNSUPPORTED, "cache dtype must be f16 or bf16");
  if (c.head_dim != 64 && c.head_dim != 128)
    return kfail(MOE_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (!power_of_two(c.page_size) || c.page_size < 16 || c.page_size > 256)
    return kfail(MOE_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
  if (c.layers <= 0 || c.pages <= 0 || c.kv_heads <= 0 || c.sequences <= 0 || c.max_blocks <= 0)
    return kfail(MOE_ERR_INVALID, "layers, pages, kv_heads, sequences and max_blocks must be positive");
  if (c.sequences > kKvMaxSeqs) return kfail(MOE_ERR_UNSUPPORTED, "more than 65536 sequences");
  if (static_cast<int64_t>(c.pages) * c.page_size > 0x7fffffffLL || c.pages > (1 << 26))
    return kfail(MOE_ERR_UNSUPPORTED, "more than 2^31 tokens or 2^26 pages");
  if (!c.k || !c.v || !c.block_table || !c.lengths || !c.refs || !c.scratch)
    return kfail(MOE_ERR_INVALID, "null pool, table, lengths, refs or scratch");
  if (misaligned16(c.k) || misaligned16(c.v)) return kfail(MOE_ERR_INVALID, "pools must be 16-byte aligned");
  const int sizes[4] = {c.layers, c.pages, c.kv_heads, c.page_size};
  for (int i = 0; i < 4; ++i) {
    const int64_t least = sizes[i] > 1 ? c.head_dim : 0;
    if (c.k_strides[i] < least || c.v_strides[i] < least || c.k_strides[i] % 8 || c.v_strides[i] % 8)
      return kfail(MOE_ERR_INVALID, "pool strides must be multiples of 8 elements, rows not overlapping");
  }
  MoeKvCache* h = new (std::nothrow) MoeKvCache();
  if (!h) return kfail(MOE_ERR_INVALID, "out of host memory");
  KvView& v = h->v;
  v.k = static_cast<char*>(c.k);
  v.v = static_cast<char*>(c.v);
  for (int i = 0; i < 4; ++i) {
    v.ks[i] = c.k_strides[i] * 2;
    v.vs[i] = c.v_strides[i] * 2;
  }
  v.layers = c.layers;
  v.pages = c.pages;
  v.heads = c.kv_heads;
  v.page = c.page_size;
  while ((1 << v.page_shift) < v.page) ++v.page_shift;
  v.hd = c.head_dim;
  v.table = c.block_table;
  v.nseq = c.sequences;
  v.max_blocks = c.max_blocks;
  v.len = c.lengths;
  v.refs = c.refs;
  int* w = static_cast<int*>(c.scratch);
  const size_t cap = std::max(c.pages, c.sequences);
  v.err = w;
  v.count = w + 1;
  v.ok = w + 2;
  v.src = w + 16;
  v.dst = v.src + cap;
  v.rows = v.dst + cap;
  v.list = v.rows + cap;
  v.off = v.list + c.pages;
  h->bf16 = c.dtype == MOE_KV_BF16;
  h->device = c.device;
  int sms = 0;
  h->num_sms = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c.device) == cudaSuccess && sms > 0
                   ? std::min(sms, kKvMaxSms) : 148;
  std::string err;
  if (!make_tmap_pool(&h->tk, c.k, h->bf16, v, v.ks, &err) ||
      !make_tmap_pool(&h->tv, c.v, h->bf16, v, v.vs, &err)) {
    delete h;
    return kfail(MOE_ERR_CUDA, err);
  }
  *out = h;
  return MOE_OK;
}

int moe_kv_destroy(MoeKvCache* cache) {
  delete cache;
  return MOE_OK;
}

int moe_kv_reserve(MoeKvCache* cache, const int32_t* seqs, const int32_t* counts, int32_t n,
                   void* stream) {
  MOE_KV_ENTER(cache);
  if (n < 0 || n > cache->v.nseq) return kfail(MOE_ERR_INVALID, "n outside [0, sequences]");
  if (n == 0) return MOE_OK;
  if (!seqs || !counts) return kfail(MOE_ERR_INVALID, "null seqs / counts");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  MOE_KV_CUDA(pdl_launch(kv_reserve_kernel, dim3(1), dim3(kPlanThreads), bitmap_bytes(cache->v), s,
                         cache->v, seqs, counts, n));
  MOE_KV_CUDA(pdl_launch(kv_copy_kernel, copy_grid(cache), dim3(256), 0, s, cache->v, cache->v,
                         static_cast<const int*>(cache->v.rows)));
  return MOE_OK;
}

int moe_kv_fork(MoeKvCache* cache, const int32_t* parents, const int32_t* children, int32_t n,
                void* stream) {
  MOE_KV_ENTER(cache);
  if (n < 0 || n > cache->v.nseq) return kfail(MOE_ERR_INVALID, "n outside [0, sequences]");
  if (n == 0) return MOE_OK;
  if (!parents || !children) return kfail(MOE_ERR_INVALID, "null parents / children");
  MOE_KV_CUDA(pdl_launch(kv_fork_kernel, dim3(std::min(n, cache->num_sms * 8)), dim3(256),
                         bitmap_bytes(cache->v), static_cast<cudaStream_t>(stream), cache->v,
                         parents, children, n));
  return MOE_OK;
}

int moe_kv_truncate(MoeKvCache* cache, const int32_t* seqs, const int32_t* lengths, int32_t n,
                    void* stream) {
  MOE_KV_ENTER(cache);
  if (n < 0 || n > cache->v.nseq) return kfail(MOE_ERR_INVALID, "n outside [0, sequences]");
  if (n == 0) return MOE_OK;
  if (!seqs || !lengths) return kfail(MOE_ERR_INVALID, "null seqs / lengths");
  MOE_KV_CUDA(pdl_launch(kv_truncate_kernel, dim3(std::min(n, cache->num_sms * 8)), dim3(256),
                         bitmap_bytes(cache->v), static_cast<cudaStream_t>(stream), cache->v, seqs,
                         lengths, n));
  return MOE_OK;
}

int moe_kv_copy_pages(MoeKvCache* cache, const int32_t* src, const int32_t* dst, int32_t n,
                      void* stream) {
  MOE_KV_ENTER(cache);
  if (n < 0 || n > cache->v.pages) return kfail(MOE_ERR_INVALID, "n outside [0, pages]");
  if (n == 0) return MOE_OK;
  if (!src || !dst) return kfail(MOE_ERR_INVALID, "null src / dst");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  MOE_KV_CUDA(pdl_launch(kv_copy_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, cache->v, src, dst, n));
  MOE_KV_CUDA(pdl_launch(kv_copy_kernel, copy_grid(cache), dim3(256), 0, s, cache->v, cache->v,
                         static_cast<const int*>(nullptr)));
  return MOE_OK;
}

int moe_kv_compact(MoeKvCache* cache, MoeKvCache* into, void* stream) {
  MOE_KV_ENTER(cache);
  const bool in_place = !into || into == cache;
  const MoeKvCache* to = in_place ? cache : into;
  const KvView &a = cache->v, &b = to->v;
  if (!in_place) {
    if (to->device != cache->device || to->bf16 != cache->bf16 || a.layers != b.layers ||
        a.heads != b.heads || a.page != b.page || a.hd != b.hd)
      return kfail(MOE_ERR_INVALID, "the two caches differ in device, dtype or page shape");
    if (b.nseq < a.nseq || b.max_blocks < a.max_blocks)
      return kfail(MOE_ERR_INVALID, "the other cache's block table is smaller");
    if (a.k == b.k || a.v == b.v || a.table == b.table || a.len == b.len || a.refs == b.refs ||
        a.err == b.err)
      return kfail(MOE_ERR_INVALID, "the two caches share memory");
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  MOE_KV_CUDA(pdl_launch(kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a,
                         in_place ? 0 : b.pages));
  MOE_KV_CUDA(pdl_launch(kv_copy_kernel, copy_grid(cache), dim3(256), 0, s, a, b,
                         static_cast<const int*>(nullptr)));
  const int64_t cells = static_cast<int64_t>(b.nseq) * b.max_blocks + b.pages;
  MOE_KV_CUDA(pdl_launch(kv_compact_tables_kernel,
                         dim3(static_cast<int>(std::min<int64_t>((cells + 255) / 256, cache->num_sms * 8))),
                         dim3(256), 0, s, a, b, in_place ? 1 : 0));
  return MOE_OK;
}

int moe_kv_append(MoeKvCache* cache, int32_t layer, const void* k, const void* v,
                  int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                  const int32_t* seqs, const int32_t* q_start, int32_t n_seqs, int32_t rows,
                  void* stream) {
  MOE_KV_ENTER(cache);
  if (const int rc = check_batch(cache, layer, seqs, q_start, n_seqs, rows)) return rc;
  if (n_seqs == 0 || rows == 0) return MOE_OK;
  if (!k || !v) return kfail(MOE_ERR_INVALID, "null k / v");
  const int64_t ks[2] = {k_token, k_head}, vs[2] = {v_token, v_head};
  if (misaligned16(k) || misaligned16(v) || bad_strides(ks) || bad_strides(vs))
    return kfail(MOE_ERR_INVALID, "k and v must be 16-byte aligned, with strides that are multiples of 8");
  const KvBatch b{seqs, q_start, n_seqs, rows};
  MOE_KV_CUDA(kv_launch_append(cache->v, b, layer, k, v, ks, vs, cache->num_sms,
                               static_cast<cudaStream_t>(stream)));
  return MOE_OK;
}

uint64_t moe_kv_attend_workspace_bytes(const MoeKvCache* cache, int32_t heads, int32_t rows,
                                       int32_t n_seqs) {
  if (!cache || heads <= 0 || rows <= 0 || n_seqs <= 0) return 0;
  return kv_attend_workspace(cache->v, heads, rows, n_seqs, cache->num_sms);
}

int moe_kv_attend(MoeKvCache* cache, const MoeKvAttendArgs* args, void* workspace,
                  uint64_t workspace_bytes, void* stream) {
  MOE_KV_ENTER(cache);
  if (!args) return kfail(MOE_ERR_INVALID, "null arguments");
  const MoeKvAttendArgs& a = *args;
  if (const int rc = check_batch(cache, a.layer, a.seqs, a.q_start, a.n_seqs, a.rows)) return rc;
  if (a.heads <= 0 || a.heads % cache->v.heads)
    return kfail(MOE_ERR_INVALID, "heads must be a positive multiple of the cache's kv_heads");
  if (!(a.scale > 0.f) || !(a.scale < 3.0e38f)) return kfail(MOE_ERR_INVALID, "scale must be positive and finite");
  if (a.n_seqs == 0 || a.rows == 0) return MOE_OK;
  if (!a.q || !a.out) return kfail(MOE_ERR_INVALID, "null q / out");
  if (misaligned16(a.q) || misaligned16(a.out) || bad_strides(a.q_strides) || bad_strides(a.out_strides))
    return kfail(MOE_ERR_INVALID, "q and out must be 16-byte aligned, with strides that are multiples of 8");
  if (static_cast<int64_t>(a.rows) * (a.heads / cache->v.heads) > 0x7fffffffLL)
    return kfail(MOE_ERR_UNSUPPORTED, "more than 2^31 query rows of one kv head");
  const size_t need = kv_attend_workspace(cache->v, a.heads, a.rows, a.n_seqs, cache->num_sms);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return kfail(MOE_ERR_WORKSPACE, "workspace must be a 256-byte aligned device pointer");
  if (workspace_bytes < need) return kfail(MOE_ERR_WORKSPACE, "workspace too small");
  const KvBatch b{a.seqs, a.q_start, a.n_seqs, a.rows};
  KvAttend k{};
  k.q = a.q;
  k.out = a.out;
  k.lse = a.lse;
  for (int i = 0; i < 2; ++i) {
    k.qs[i] = a.q_strides[i];
    k.os[i] = a.out_strides[i];
    k.ls[i] = a.lse_strides[i];
  }
  k.heads = a.heads;
  k.layer = a.layer;
  k.scale = a.scale;
  MOE_KV_CUDA(kv_launch_attend(cache->v, cache->tk, cache->tv, cache->bf16, b, k, workspace,
                               cache->num_sms, static_cast<cudaStream_t>(stream)));
  return MOE_OK;
}

int moe_kv_status(MoeKvCache* cache, void* stream) {
  MOE_KV_ENTER(cache);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int code = 0;
  MOE_KV_CUDA(cudaMemcpyAsync(&code, cache->v.err, sizeof(int), cudaMemcpyDeviceToHost, s));
  MOE_KV_CUDA(cudaMemsetAsync(cache->v.err, 0, sizeof(int), s));
  MOE_KV_CUDA(cudaStreamSynchronize(s));
  switch (code) {
    case DEV_OK: return MOE_OK;
    case DEV_BAD_SEQ:
      return kfail(MOE_ERR_INVALID, "a sequence index is out of range, or the same sequence came twice "
                                    "where it is written");
    case DEV_BAD_LENGTH:
      return kfail(MOE_ERR_INVALID, "a length does not fit: a child that is not empty, a longer new length, "
                                    "more tokens than the block table holds, more new rows than tokens, or "
                                    "offsets of rows that decrease or leave the rows");
    case DEV_BAD_PAGE:
      return kfail(MOE_ERR_INVALID, "a page is out of range or missing from the block table, or a copied "
                                    "page came twice");
    case DEV_NO_PAGES: return kfail(MOE_ERR_NO_PAGES, "the pool has too few free pages");
    default: break;
  }
  if (code >= DEV_TIMEOUT_FULL && code <= DEV_TIMEOUT_CONV)
    return kfail(MOE_ERR_TIMEOUT, "an attention wait ran out of time (code " + std::to_string(code) + ")");
  return kfail(MOE_ERR_DEVICE, "a cache kernel reported device error code " + std::to_string(code));
}

}  // extern "C"
