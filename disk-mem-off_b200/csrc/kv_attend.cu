// Attention of new tokens over the paged K/V cache (moe_kv_attend):
//
//   s_j = scale * q . k_j  for the tokens j up to the row's own position
//   o   = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
//
// in one pass over the keys with the running maximum and sum in fp32.
//
// Rows.  The `group` query heads that share a kv head read the same keys, so a row is
// one (new token, head of the group) pair and an entry of m tokens has m * group rows
// of each kv head.  128 rows fill the M of one tcgen05.mma.
//
// Work.  kv_plan_kernel (one CTA) cuts the entries into units: 256 rows that two
// warpgroups work on against the same keys ("pair"), 33 to 128 rows that one warpgroup
// works on alone ("single": the ends of chunks), or up to 32 ("few": decode steps).  A
// unit of one kv head costs its number of 64-key tiles and a constant.  All units, pairs
// first and counted twice since they take both warpgroups, are laid on one line that is
// cut into equal shares, one for each SM, so the load is even for any mix of lengths and
// an SM meets one or two kinds; a unit cut by a share's border leaves fp32 partial
// results that kv_merge_kernel joins in share order (same bits every time).
//
// kv_attend_kernel (one CTA an SM, 384 threads): warps 0-3 and 4-7 are the two softmax
// warpgroups, a thread a row; warp 8 fetches K and V tiles page by page (TMA, 128-byte
// swizzle) into one ring, warp 11 the Q tiles; warps 9 and 10 issue S = Q K^T (both
// operands in shared memory, K major) and O += P V (P from TMEM, V as an N-major operand,
// so that V needs no transposed copy), one for each softmax warpgroup: a single issuing
// warp took 2,590 cycles for a tile of both, most of them between the products.  TMEM: two
// S buffers of 64 keys for each warpgroup (P overwrites its S) and its O, 512 columns in
// all.  S runs two tiles ahead of the product with V, so the softmax finds its next S
// ready.  (Tiles of 128 keys leave no room for a second S buffer; with one, 64-wide heads
// took 51 us instead of 40.)  Every wait is bounded.
//
// What bounds it (device time).  Decode: the reading of K and V (2 x 131071 tokens: 1.07 GB
// in 186 us, 5.8 TB/s).  Chunks: of the 1,940 cycles that 64 keys of a pair take, starts and
// ends of units included, the tensor cores have 1,280 and the special-function units 1,024,
// and the clock falls to about 1.4 GHz under the power limit (4096 new on 4096 cached
// tokens: 1.24 ms, 1.0 PFLOP/s; a polynomial in place of every eighth to every second
// exponential: no gain, then a loss).  Short units: instructions that run once a unit, in
// two warps a scheduler.
//
// Roundings.  Scores, maxima, sums and O are fp32.  The probabilities are rounded once, to
// the cache's 16-bit type, since both operands of the product with V have one type: half a
// step, 2^-11 or 2^-8 relative (the sum takes them unrounded).  The result is rounded to
// that type once.
#include <cuda_bf16.h>
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kv_internal.h"

namespace moe {

constexpr int kTile = 128;       // rows of a warpgroup
constexpr int kKeys = 64;        // keys of a tile
constexpr int kPlanT = 1024;     // threads of the plan kernel
constexpr int kPlanSmem = 512;   // units of a list whose prefix sums fit its shared memory

// Rows [r0, r0 + rows) of an entry, for every kv head.
struct KaUnit {
  int seq;    // -1: not a sequence (rows of zeros)
  int row0;   // the entry's first row in q / out
  int r0;     // first packed row (token * group + head of the group)
  int rows;
  int base;   // position of the entry's first new token (may be negative: sees nothing)
  int len;    // tokens of the sequence
  int tiles;  // key tiles that the last row needs
  int pad;
};
static_assert(sizeof(KaUnit) == 32, "two 16-byte loads");

// A share: `count` tiles from tile `tile` of kv head `head` of list entry `item` on.
struct KaStart {
  int item, head, tile, count;
};
// A unit that the ends of shares cut: its pieces lie in shares first .. last.
struct KaMerge {
  int kind, first, last, head;
  int item, pad[3];
};
static_assert(sizeof(KaStart) == 16 && sizeof(KaMerge) == 32, "16-byte loads");
constexpr int kMergeRows = 16;

// Kinds of units: rows of a unit, shares an SM.
constexpr int kPair = 0, kSingle = 1, kFew = 2, kKinds = 3;
constexpr int kFewRows = 32;
// What beginning and ending a unit costs, in tiles of its kind (64 decode contexts of
// 1 to 8192 tokens: 64 us with 2, 58 with 3, 55 with 5; 33 mixed chunks: 170 with 3, 178
// with 8).
__host__ __device__ constexpr int kind_extra(int k) { return k == kPair ? 3 : k == kSingle ? 4 : 5; }
// The least cost worth a warpgroup of its own.
constexpr int kLeastShare = 2;
__host__ __device__ constexpr int kind_rows(int k) { return k == kPair ? 2 * kTile : k == kSingle ? kTile : kFewRows; }
__host__ __device__ constexpr int kind_shares(int k) { return k == kPair ? 1 : 2; }

struct KaWs {
  size_t start[kKinds], list[kKinds], pre[kKinds], o[kKinds], ml[kKinds], merge, n_merge, total;
  int cap[kKinds];
};

static KaWs ka_ws(const KvView& c, int heads, int rows, int n, int num_sms) {
  KaWs w{};
  size_t o = 0;
  auto take = [&](size_t b) {
    const size_t at = o;
    o = (o + b + 255) & ~size_t(255);
    return at;
  };
  const int64_t packed = static_cast<int64_t>(rows) * (heads / c.heads);
  size_t merges = 0;
  w.cap[0] = packed > kTile ? static_cast<int>(packed / (2 * kTile) + std::min<int64_t>(n, packed / kTile)) : 0;
  w.cap[1] = packed > kFewRows ? n : 0;
  w.cap[2] = n;
  for (int k = 0; k < kKinds; ++k) {
    const size_t shares = static_cast<size_t>(num_sms) * kind_shares(k);
    const size_t prow = 2 * shares * (w.cap[k] ? kind_rows(k) : 0);
    w.start[k] = take(shares * sizeof(KaStart));
    w.list[k] = take(static_cast<size_t>(w.cap[k]) * sizeof(KaUnit));
    w.pre[k] = take((static_cast<size_t>(w.cap[k]) + 1) * 8);
    w.o[k] = take(prow * c.hd * 4);
    w.ml[k] = take(prow * 8);
    merges += shares;
  }
  w.merge = take(merges * sizeof(KaMerge));
  w.n_merge = take(4);
  w.total = o;
  return w;
}

size_t kv_attend_workspace(const KvView& c, int heads, int rows, int n_seqs, int num_sms) {
  return ka_ws(c, heads, rows, n_seqs, num_sms).total;
}

// The workspace by kind (kPair, kSingle, kFew), for the kernels.
struct KaList {
  KaStart* start;
  KaUnit* list;
  long long* pre;
  float* o;    // [share][0 its first unit, 1 its last][rows][hd] unnormalised
  float2* ml;  // running maximum (base 2, scaled) and sum of the same rows
};
struct KaPtrs {
  KaList pair, single, few;
  KaMerge* merge;
  int* n_merge;
  MOE_DEV KaList kind(int k) const { return k == kPair ? pair : k == kSingle ? single : few; }
};

// ------------------------------------------------------------------ plan
// Inclusive sums of N numbers over the plan CTA, in place; total gets the whole sums.
// `busy`: the warps that may hold anything but zero.
template <int N>
MOE_DEV void plan_scan(long long (&v)[N], int busy, long long (&total)[N]) {
  __shared__ long long part[N][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp < busy) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const long long u = __shfl_up_sync(0xffffffffu, v[k], o);
        if (lane >= o) v[k] += u;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (lane == 31) part[k][warp] = v[k];
  }
  __syncthreads();
  long long p[N];
#pragma unroll
  for (int k = 0; k < N; ++k) p[k] = lane < busy ? part[k][lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (o >= busy) break;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long long u = __shfl_up_sync(0xffffffffu, p[k], o);
      if (lane >= o) p[k] += u;
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    total[k] = __shfl_sync(0xffffffffu, p[k], busy - 1);
    const long long before = __shfl_sync(0xffffffffu, p[k], max(min(warp, busy) - 1, 0));
    if (warp) v[k] += before;
  }
  __syncthreads();  // part is written again by the next call
}

MOE_DEV int key_tiles(int base, int last_token) {
  // tokens visible to the unit's last row, at least one tile (rows that see nothing still
  // have to be written).  So only the last tile holds keys past the sequence's end, with
  // fewer tokens than new rows (base < 0) too: the MMA warps rely on it when they clear V.
  const long long vis = max(static_cast<long long>(base) + last_token + 1, 1ll);
  return static_cast<int>((vis + kKeys - 1) / kKeys);
}

// Where the cost w0 lies in a list whose prefix sums (of one kv head) are pre[0 .. n]; T:
// 32 bits when every cost fits.  A unit's extra comes before its tiles, so a border
// inside it leaves the unit whole.
struct KaPlace {
  int item, head, tile;
  long long unit;   // the unit's cost begins here
  long long cost;   // and is this
  long long tiles;  // tiles before w0
};
// One kind's part of the line: pairs from 0 on, the others after `before`.  CTA c has
// [2 per c, 2 per (c + 1)) of the line; a pair unit takes two of it for one of cost, and the
// other kinds' part of a CTA is halved between its warpgroups.
struct KaLine {
  long long per, before, all;
  bool small, pair;
  MOE_DEV void range(int share, long long* w0, long long* w1) const {
    if (pair) {
      *w0 = min(share * per, all);
      *w1 = min((share + 1) * per, all);
      return;
    }
    const long long at = 2 * per * (share >> 1) - before;
    const long long lo = min(max(at, 0ll), all), hi = min(max(at + 2 * per, 0ll), all);
    const long long mid = lo + ((hi - lo + 1) >> 1);
    *w0 = share & 1 ? mid : lo;
    *w1 = share & 1 ? hi : mid;
  }
  MOE_DEV int share_of(long long pos) const {
    const long long at = pair ? pos : pos + before, len = pair ? per : 2 * per;
    const int c = small ? static_cast<int>(static_cast<uint32_t>(at) / static_cast<uint32_t>(len))
                        : static_cast<int>(at / len);
    if (pair) return c;
    long long w0, w1;
    range(2 * c, &w0, &w1);
    return 2 * c + (pos >= w1 ? 1 : 0);
  }
};

template <typename T>
MOE_DEV KaPlace plan_place(const long long* pre, int n, T w0, int heads, int extra) {
  int lo = 0, hi = n;  // heads * pre[lo] <= w0 < heads * pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (static_cast<T>(pre[mid]) * heads <= w0) lo = mid;
    else hi = mid;
  }
  const T base = static_cast<T>(pre[lo]) * heads, cost = static_cast<T>(pre[lo + 1] - pre[lo]);
  const T r = w0 - base, head = r / cost, at = r - head * cost;
  KaPlace p;
  p.item = lo;
  p.head = static_cast<int>(head);
  p.tile = at > static_cast<T>(extra) ? static_cast<int>(at) - extra : 0;
  p.unit = static_cast<long long>(base + head * cost);
  p.cost = static_cast<long long>(cost);
  p.tiles = p.unit - (static_cast<long long>(lo) * heads + p.head) * extra + p.tile;
  return p;
}

// (1) entries -> units and the prefix sums of their costs, (2) each share's first tile and
// the units that the shares' ends cut.  One CTA: two dependent loads, two scans, a search.
__global__ void __launch_bounds__(kPlanT) kv_plan_kernel(const KvView c, const KvBatch b,
                                                         const int group, const int num_sms,
                                                         const KaPtrs w, const int cap0) {
  pdl_enter();
  __shared__ long long spre[kKinds][kPlanSmem + 1];
  __shared__ int s_merges;
  __shared__ long long s_tiles[kPlanT];
  __shared__ int4 s_entry[kPlanT];       // the chunk's entries: seq, row0, m, len
  __shared__ int s_pairs[kPlanT + 1];    // pairs before each of them
  const int tid = threadIdx.x;
  if (tid == 0) s_merges = 0;
  // (1)
  int n_pair = 0, n_single = 0, n_few = 0;
  long long work_pair = 0, work_single = 0, work_few = 0;  // of one kv head
  bool bad = false;
  long long* pre_pair = cap0 <= kPlanSmem ? spre[0] : w.pair.pre;
  long long* pre_single = b.n <= kPlanSmem ? spre[1] : w.single.pre;
  long long* pre_few = b.n <= kPlanSmem ? spre[2] : w.few.pre;
  for (int i0 = 0; i0 < b.n; i0 += kPlanT) {
    const int i = i0 + tid, busy = min((b.n - i0 + 31) / 32, 32);
    int seq = -1, row0 = 0, m = 0, len = 0;
    if (i < b.n) {
      seq = b.seqs[i];
      row0 = b.q_start[i];
      const long long end = b.q_start[i + 1];
      if (row0 < 0 || end < row0 || end > b.rows) {
        record_error(c.err, DEV_BAD_LENGTH);
        bad = true;
      } else {
        m = static_cast<int>(end) - row0;
      }
      if (seq < 0 || seq >= c.nseq) {
        if (m > 0) record_error(c.err, DEV_BAD_SEQ);
        seq = -1;
      } else {
        len = max(c.len[seq], 0);
        if (len > static_cast<long long>(c.max_blocks) << c.page_shift) {
          record_error(c.err, DEV_BAD_LENGTH);
          len = c.max_blocks << c.page_shift;
        }
      }
    }
    const int rows = m * group;
    const int rem = rows & (2 * kTile - 1);
    const int na = rows / (2 * kTile) + (rem > kTile ? 1 : 0);
    const bool single = rem > kFewRows && rem <= kTile, few = rem > 0 && rem <= kFewRows;
    const int tiles = key_tiles(len - m, m - 1);
    // few and single: counts (at most 1024) in the high bits, costs in the low 44; pairs
    const KaUnit rest{seq, row0, rows - rem, rem, len - m, len, tiles, 0};
    constexpr long long kOne = 1ll << 44, kLow = kOne - 1;
    long long at[3] = {few ? kOne + tiles + kind_extra(kFew) : 0, single ? kOne + tiles + kind_extra(kSingle) : 0, na};
    long long total[3];
    plan_scan(at, busy, total);
    if (few) {
      const int j = n_few + static_cast<int>(at[0] >> 44) - 1;
      w.few.list[j] = rest;
      pre_few[j + 1] = work_few + (at[0] & kLow);
    }
    if (single) {
      const int j = n_single + static_cast<int>(at[1] >> 44) - 1;
      w.single.list[j] = rest;
      pre_single[j + 1] = work_single + (at[1] & kLow);
    }
    n_few += static_cast<int>(total[0] >> 44);
    work_few += total[0] & kLow;
    n_single += static_cast<int>(total[1] >> 44);
    work_single += total[1] & kLow;
    if (total[2] == 0) continue;
    s_entry[tid] = make_int4(seq, row0, m, len);
    s_pairs[tid + 1] = static_cast<int>(at[2]);
    if (tid == 0) s_pairs[0] = 0;
    __syncthreads();
    const int pairs = min(static_cast<int>(total[2]), cap0 - n_pair);
    for (int j0 = 0; j0 < pairs; j0 += kPlanT) {  // a thread a pair
      const int j = j0 + tid;
      long long sum[1] = {0}, all[1];
      KaUnit u{};
      if (j < pairs) {
        int lo = 0, hi = min(b.n - i0, kPlanT);  // s_pairs[lo] <= j < s_pairs[hi]
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_pairs[mid] <= j) lo = mid;
          else hi = mid;
        }
        const int4 e = s_entry[lo];
        const int r0 = (j - s_pairs[lo]) * 2 * kTile, r1 = min(r0 + 2 * kTile, e.z * group);
        u = KaUnit{e.x, e.y, r0, r1 - r0, e.w - e.z, e.w, key_tiles(e.w - e.z, (r1 - 1) / group), 0};
        w.pair.list[n_pair + j] = u;
        sum[0] = u.tiles + kind_extra(kPair);
      }
      plan_scan(sum, min((pairs - j0 + 31) / 32, 32), all);
      if (j < pairs) pre_pair[n_pair + j + 1] = work_pair + sum[0];
      work_pair += all[0];
    }
    n_pair += pairs;
  }
  if (tid == 0) pre_pair[0] = pre_single[0] = pre_few[0] = 0;
  // offsets that decrease can give a row to two entries: none is worked on then
  if (__syncthreads_or(bad)) {
    n_pair = n_single = n_few = 0;
    work_pair = work_single = work_few = 0;
  }
  // (2) a thread for each share of each kind
  const int k = tid < num_sms ? kPair : tid < 3 * num_sms ? kSingle : kFew;
  const int share = tid - (k == kPair ? 0 : k == kSingle ? num_sms : 3 * num_sms);
  const bool mine = share < num_sms * kind_shares(k);
  const int extra = kind_extra(k);
  const int n = k == kPair ? n_pair : k == kSingle ? n_single : n_few;
  const long long* pre = k == kPair ? pre_pair : k == kSingle ? pre_single : pre_few;
  const long long cost_pair = work_pair * c.heads, cost_single = work_single * c.heads, cost_few = work_few * c.heads;
  const long long line = 2 * cost_pair + cost_single + cost_few;
  KaLine l;
  l.small = line < 0x40000000;
  const int halves = 2 * num_sms;
  l.per = max(l.small ? (static_cast<int>(line) + halves - 1) / halves : (line + halves - 1) / halves,
              static_cast<long long>(kLeastShare));
  l.pair = k == kPair;
  l.before = k == kPair ? 0 : k == kSingle ? 2 * cost_pair : 2 * cost_pair + cost_single;
  l.all = k == kPair ? cost_pair : k == kSingle ? cost_single : cost_few;
  long long w0, w1;
  l.range(share, &w0, &w1);
  KaPlace p{};
  p.tiles = l.all - static_cast<long long>(n) * extra * c.heads;
  if (mine && w0 < l.all)
    p = l.small ? plan_place<uint32_t>(pre, n, static_cast<uint32_t>(w0), c.heads, extra)
                : plan_place<unsigned long long>(pre, n, static_cast<unsigned long long>(w0), c.heads, extra);
  s_tiles[tid] = p.tiles;  // the next share begins where this one ends
  __syncthreads();
  if (mine) {
    const KaList list = w.kind(k);
    const long long end = share + 1 < num_sms * kind_shares(k)
                              ? s_tiles[tid + 1] : l.all - static_cast<long long>(n) * extra * c.heads;
    list.start[share] = KaStart{p.item, p.head, p.tile, static_cast<int>(end - p.tiles)};
    // a unit that is cut here first: its first tile lies in the share that ends here
    if (w0 < w1 && p.tile > 0) {
      const int first = l.share_of(p.unit + extra);
      long long f0, f1;
      l.range(first, &f0, &f1);
      if (f1 == w0)
        w.merge[atomicAdd(&s_merges, 1)] =
            KaMerge{k, first, l.share_of(p.unit + p.cost - 1), p.head, p.item, {0, 0, 0}};
    }
  }
  __syncthreads();
  if (tid == 0) *w.n_merge = s_merges;
}
static_assert(5 * kKvMaxSms <= kPlanT, "a thread for each share");

// ------------------------------------------------------------------ the kernel
template <int HD>
struct KaCfg {
  static constexpr int kQ = kTile * HD * 2;      // one warpgroup's Q tile
  static constexpr int kStage = kKeys * HD * 2;  // one K or V tile
  static constexpr int kStages = HD == 128 ? 10 : 16;
  static constexpr int kHalf = kStages / 2;  // of each of the two rings of the other kinds
  static constexpr int kLoads = HD / 64;          // 64-dim blocks of a tile
  // barriers, and the 8 warps' (max, sum) of 16 rows each
  static constexpr size_t kSmem = 1024 + 2 * kQ + kStages * kStage + 768 + 1024;
};
static_assert(KaCfg<128>::kSmem <= 227 * 1024 && KaCfg<64>::kSmem > 114 * 1024,
              "one CTA, and with it all of TMEM, an SM");

// Twelve warps (8: K / V, 9 and 10: MMA, 11: Q, then K / V), so that each third is a warpgroup and
// registers can move between them: 384 * 168 at launch = 2 * 128 * 208 + 128 * 80 + rest.
constexpr int kAttThreads = 384;
constexpr int kRegsSoftmax = 208, kRegsOther = 80;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kAttThreads * 168, "more than the launch had");
template <int N>
MOE_DEV void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
MOE_DEV void regs_fewer() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr uint32_t kOCols = 256;  // TMEM: S of stream s, buffer b at s * 128 + b * 64; O at 256 + s * 128

// Five-dimensional tiled load (dim, row, head, page, layer); a page past the end reads
// as zeros.
MOE_DEV void tma_load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4,
                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4),
      "r"(smem_u32(bar))
      : "memory");
}

MOE_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
MOE_DEV void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Instruction descriptor of f16 (fmt 0) or bf16 (1) operands, M = 128, B K-major or (nmajor) N-major.
__host__ __device__ constexpr uint32_t ka_idesc(uint32_t fmt, int n, uint32_t nmajor) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (nmajor << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTile >> 4) << 24);
}

// Descriptor of a V tile as the N-major B operand: rows of a key with 64 dims (128
// bytes, 128-byte swizzle), 8 keys every 1024 bytes (SBO), the next 64 dims 8 KiB on (LBO).
MOE_DEV uint64_t nmajor_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(kKeys * 128 >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// The tiles of a share in order.
struct KaCursor {
  const KaUnit* list;
  KaUnit u;
  int item, head, tile, left, heads;
  MOE_DEV void load() {
    const int4* p = reinterpret_cast<const int4*>(list + item);
    const int4 a = p[0], b = p[1];
    u.seq = a.x; u.row0 = a.y; u.r0 = a.z; u.rows = a.w;
    u.base = b.x; u.len = b.y; u.tiles = b.z;
  }
  MOE_DEV static int4 start(const KaPtrs& w, int kind, int share) {
    return *reinterpret_cast<const int4*>(w.kind(kind).start + share);
  }
  MOE_DEV void init(const KaPtrs& w, int kind, const int4 s, int kv_heads) {
    list = w.kind(kind).list;
    item = s.x;
    head = s.y;
    tile = s.z;
    left = s.w;
    heads = kv_heads;
    if (left > 0) load();
  }
  // this share's last tile of the unit
  MOE_DEV bool ends_unit() const { return tile + 1 == u.tiles || left == 1; }
  MOE_DEV void next() { skip(1); }
  // the next n tiles, all of this unit
  MOE_DEV void skip(int n) {
    left -= n;
    tile += n;
    if (tile == u.tiles) {
      tile = 0;
      if (++head == heads) {
        head = 0;
        ++item;
        if (left > 0) load();
      }
    }
  }
};

// Page numbers of a sequence, 32 blocks at a time in the lanes of the producer warp,
// the next 32 already on their way.
struct KaPages {
  int seq = -2, chunk = -1, ids = -1, nxt = -1;
  MOE_DEV static int fetch(const KvView& c, const KaUnit& u, int chunk) {
    const int blk = chunk * 32 + (threadIdx.x & 31);
    const int need = (u.len + c.page - 1) >> c.page_shift;
    return u.seq >= 0 && blk < need ? c.table[static_cast<long long>(u.seq) * c.max_blocks + blk] : -1;
  }
  MOE_DEV void at(const KvView& c, const KaUnit& u, int block) {
    const int want = block >> 5;
    if (u.seq != seq || want != chunk) {
      ids = u.seq == seq && want == chunk + 1 ? nxt : fetch(c, u, want);
      nxt = fetch(c, u, want + 1);
      seq = u.seq;
      chunk = want;
    }
  }
};

// A ring of K and V tiles, filled by one warp.
struct KaRing {
  const KvView& c;
  const CUtensorMap &tk, &tv;
  const int layer;
  uint64_t *full, *empty;
  const uint32_t smem;
  const int stages, bytes, loads;
  volatile int* abort_flag;
  int st = 0, n = 0;  // next stage, tiles put
  uint32_t ph = 1;    // parity of the wait for it
  // Tile `tile` of the unit's keys or values into the next stage: boxes of up to 64 rows by
  // 64 dims, a lane each.
  MOE_DEV bool put(const KaUnit& u, int head, int tile, KaPages& pg, bool val) {
    const int lane = threadIdx.x & 31;
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], ph, abort_flag))) return false;
    const int box = min(c.page, kKeys);
    const int p = lane / loads, kb = lane - p * loads;
    const int key = tile * kKeys + p * box;
    pg.at(c, u, (tile * kKeys) >> c.page_shift);
    if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
    __syncwarp();
    const int blk = key >> c.page_shift;
    int id = __shfl_sync(0xffffffffu, pg.ids, blk & 31);
    if (p * box < kKeys) {
      if (id < 0 || id >= c.pages) {
        // past the sequence's last page: zeros; before it: a hole in the table
        if (key < u.len) record_error(c.err, DEV_BAD_PAGE);
        id = c.pages;
      }
      tma_load_5d(smem + st * bytes + kb * (kKeys * 128) + p * box * 128, val ? &tv : &tk, kb * 64,
                  key & (c.page - 1), head, id, layer, &full[st]);
    }
    ++n;
    if (++st == stages) {
      st = 0;
      ph ^= 1;
    }
    return true;
  }
  // This share's tiles of the cursor's unit, K two tiles ahead of V as the MMAs take them.
  MOE_DEV bool put_unit(KaCursor& x, KaPages& pg) {
    const int nt = min(x.left, x.u.tiles - x.tile);
    for (int j = -2; j < nt; ++j) {
      if (j >= 0 && !put(x.u, x.head, x.tile + j, pg, true)) return false;
      if (j + 2 < nt && !put(x.u, x.head, x.tile + j + 2, pg, false)) return false;
    }
    x.skip(nt);
    return true;
  }
  // All copies have landed; with `read` also waits until all stages have been let go.
  MOE_DEV void drain(bool& read) {
    const int k = min(n, stages);
    for (int i = 0; i < k; ++i) {
      if (st-- == 0) {
        st = stages - 1;
        ph ^= 1;
      }
      mbar_wait_drain(&full[st], ph ^ 1);
      if (read) read = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], ph ^ 1, abort_flag));
    }
    __syncwarp();
  }
  MOE_DEV void drain(bool&& read) {
    bool r = read;
    drain(r);
  }
};

// Up to 128 rows of a unit's Q from packed row `first` on, by a warp, swizzled as the MMA
// reads them.
template <int HD>
MOE_DEV void fetch_q(const KvAttend& a, const KaUnit& u, int head, int group, int first, uint32_t smem) {
  constexpr int ch = HD / 8, step = 32 / ch;  // 16-byte chunks of a row, rows at a time
  const int lane = threadIdx.x & 31;
  int row = lane / ch;
  const int chunk = lane - row * ch;
  const int rows = min(u.rows - first, kTile);
  const uint32_t to = smem + (chunk >> 3) * (kTile * 128);
  const int dtok = step / group, dhg = step - dtok * group;
  const int packed = u.r0 + first + row;
  const int tok = packed / group;
  int hg = packed - tok * group;
  const int64_t dwrap = a.qs[0] - group * a.qs[1], dsrc = dtok * a.qs[0] + dhg * a.qs[1];
  const __half* src = static_cast<const __half*>(a.q) + (u.row0 + static_cast<int64_t>(tok)) * a.qs[0] +
                      (static_cast<int64_t>(head) * group + hg) * a.qs[1] + chunk * 8;
#pragma unroll 8
  for (; row < rows; row += step) {
    cp_async16(to + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), src);
    src += dsrc;
    hg += dhg;
    if (hg >= group) {
      hg -= group;
      src += dwrap;
    }
  }
}

// One lane of a converged warp, the same one every time.
MOE_DEV bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// The same value in every lane, and known as such to the compiler.
MOE_DEV uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// The whole warp waits and takes the same way out.
MOE_DEV bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag));
}

template <bool BF16>
MOE_DEV uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

MOE_DEV float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 32 TMEM columns of a row on their way; they may be read after tmem_landed.
MOE_DEV void tmem_ld32_start(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// Waits for this thread's TMEM loads; v passes through, so that no use moves above.
MOE_DEV void tmem_landed(float* v, int n) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < n; ++i) asm volatile("" : "+f"(v[i]));
}
MOE_DEV void load_s(uint32_t taddr, float (&sc)[kKeys]) {
#pragma unroll
  for (int i = 0; i < kKeys / 32; ++i) tmem_ld32_start(taddr + i * 32, sc + i * 32);
  tmem_landed(sc, kKeys);
}

// ------------------------------------------------------------------ few rows
// Units of at most 32 rows (decode steps).  They are bound by the reading of K and V, and
// a tcgen05.mma of 128 rows would spend its time, and its softmax warps theirs, on padding.
// So each warpgroup works alone on 64-key tiles of its own ring: MT 16-row blocks times
// 4 / MT slices of 16 * MT keys, mma.sync m16n8k16 from the same swizzled tiles.  A warp
// keeps its own running maximum, sum and O (fp32, registers) over its slices: no exchange
// inside a unit, one join of the slices through shared memory (the idle Q tile) at its
// end, while the next tiles load and the other warpgroup computes.
MOE_DEV void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
MOE_DEV void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
MOE_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Two fp32 operations in one instruction.
MOE_DEV uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
MOE_DEV float2 split_pair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
MOE_DEV uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
MOE_DEV uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A unit cut by the ends of shares leaves a piece in each of its shares: rows
// unnormalised in fp32 with their maximum (base 2, scaled) and sum, in the share's slot 0
// (the unit began in an earlier share) or 1 (it goes on in a later one).  A maximum of -inf
// is kept for rows that see no token at all: the merge tells them by it.
MOE_DEV float2 piece_ml(float top, float sum, bool sees) {
  return make_float2(sees ? fmaxf(top, -FLT_MAX) : -INFINITY, sum);
}
MOE_DEV long long piece_slot(int kind, int share, bool tail, int row) {
  return (2ll * share + (tail ? 1 : 0)) * kind_rows(kind) + row;
}

MOE_DEV void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Results of one row and head: lane's HD / 32 values, the log of the sum.  Whether the row
// sees a token is told by its position, not by the sum: scores of NaN or of -inf alone leave
// no maximum either, and give NaN.
template <int HD, bool BF16>
MOE_DEV void write_row(const KvAttend& a, long long row, int h, const float* v, float top, float sum, bool sees) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  const float inv = 1.f / sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<__half*>(a.out) + row * a.os[0] + h * a.os[1]) + lane * (V / 2);
#pragma unroll
  for (int e = 0; e < V / 2; ++e) dst[e] = sees ? pack2<BF16>(v[2 * e] * inv, v[2 * e + 1] * inv) : 0u;
  if (a.lse && lane == 0)
    a.lse[row * a.ls[0] + h * a.ls[1]] = sees ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

template <int HD, bool BF16>
struct KaFew {
  using C = KaCfg<HD>;
  const KvView& c;
  const KvAttend& a;
  const KaPtrs& w;
  const int group;
  const float scale_log2;
  uint8_t *sQ, *sR;  // this warpgroup's Q tile and ring
  uint64_t *full, *empty, *joined;
  float2* s_ml;  // [4][16]
  volatile int* abort_flag;
  int n = 0;      // ring tiles taken
  int units = 0;  // joins so far
  uint32_t next_q[HD / 16][4];  // Q fragments of the next unit
  int next_seen[2];             // tokens that its rows see
  // Row `lane` of the unit, the next one's and the current one's: token of the batch and
  // head of its group.  A division, made once for all kv heads of an entry.
  int rows_of = -1;  // list entry of the next unit
  int next_tok, next_hg, next_sees;
  int tok, hg;  // ~hg: the row sees no token

  // Q fragments of rows mi * 16 + g and + 8 of the cursor's unit, and the tokens they see
  MOE_DEV void fetch_q(const KaCursor& x) {
    const KaUnit& u = x.u;
    const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (rows_of != x.item) {
      rows_of = x.item;
      const int packed = u.r0 + min(lane, u.rows - 1);
      const int k = packed / group;
      next_hg = packed - k * group;
      next_tok = u.row0 + k;
      next_sees = lane < u.rows ? max(min(u.base + k + 1, u.len), 0) : 0;
    }
    const long long at = next_tok * a.qs[0] + (static_cast<long long>(x.head) * group + next_hg) * a.qs[1];
    const int first = u.rows <= 16 ? 0 : (warp >> 1) * 16;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int pr = first + g + 8 * r;
      next_seen[r] = __shfl_sync(0xffffffffu, next_sees, pr);
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const __half*>(a.q) +
                                                              __shfl_sync(0xffffffffu, at, pr));
      const bool valid = pr < u.rows;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        next_q[k][r] = valid ? src[k * 8 + t] : 0u;
        next_q[k][r + 2] = valid ? src[k * 8 + t + 4] : 0u;
      }
    }
  }

  // One unit, or this share's piece of it; false when a wait ran out.
  template <int MT>
  MOE_DEV bool unit(KaCursor& x, int share) {
    constexpr float shift = BF16 ? 0.f : 7.f;  // as in the softmax warpgroups
    constexpr int kSlices = 4 / MT, kKeysW = 16 * MT;  // keys of a warp
    const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
    const int slice = warp % kSlices;  // of 16-row block warp / kSlices
    const int g = lane >> 2, t = lane & 3;
    const KaUnit u = x.u;
    const int head = x.head;
    const bool cut_front = x.tile > 0;
    uint32_t q[HD / 16][4];
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[k][e] = next_q[k][e];
    const int seen[2] = {next_seen[0], next_seen[1]};
    tok = next_tok;
    hg = next_sees > 0 ? next_hg : ~next_hg;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool whole = true, first = true;
    // lane addresses inside a 16-key group: K rows (lane >> 4) * 8 + (lane & 7), chunk
    // (lane >> 3 & 1); V rows lane & 15, chunk lane >> 4
    const int krow = slice * kKeysW + ((lane >> 4) << 3) + (lane & 7), vrow = slice * kKeysW + (lane & 15);
    for (bool ends = false; !ends;) {
      ends = x.ends_unit();
      const int key0 = x.tile * kKeys;
      if (ends) whole = x.tile + 1 == u.tiles;
      x.next();
      // S = Q K^T of this warp's slice
      int st = n % C::kHalf;
      if (!warp_wait(&full[st], (n / C::kHalf) & 1, abort_flag)) return false;
      uint32_t base = smem_u32(sR) + st * C::kStage + krow * 128;
      float sc[MT][2][4];
#pragma unroll
      for (int kg = 0; kg < MT; ++kg) {
#pragma unroll
        for (int i = 0; i < 2; ++i) sc[kg][i][0] = sc[kg][i][1] = sc[kg][i][2] = sc[kg][i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const int chunk = (k & 3) * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldsm4(base + kg * 2048 + (k >> 2) * 8192 + ((chunk ^ (krow & 7)) << 4), b);
          mma16816<BF16>(sc[kg][0], q[k], b[0], b[1]);
          mma16816<BF16>(sc[kg][1], q[k], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      ++n;
      // softmax of the slice
      const int slice_end = key0 + (slice + 1) * kKeysW;
      if (__any_sync(0xffffffffu, min(seen[0], seen[1]) < slice_end)) {
        const int col0 = key0 + slice * kKeysW + 2 * t;
#pragma unroll
        for (int kg = 0; kg < MT; ++kg)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col0 + kg * 16 + i * 8 + (e & 1) >= seen[e >> 1]) sc[kg][i][e] = -INFINITY;
      }
      float alpha[2];
      bool grow = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int kg = 0; kg < MT; ++kg)
          top = fmaxf(top, fmaxf(fmaxf(sc[kg][0][2 * r], sc[kg][0][2 * r + 1]),
                                 fmaxf(sc[kg][1][2 * r], sc[kg][1][2 * r + 1])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * scale_log2;
        alpha[r] = 1.f;
        if (top - m[r] > 8.f) {
          alpha[r] = exp2_ftz(m[r] - top);
          m[r] = top;
          grow = true;
        }
        const float ref = m[r] == -INFINITY ? 0.f : m[r] - shift;
        float sum = 0.f;
#pragma unroll
        for (int kg = 0; kg < MT; ++kg)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 2 * r; e < 2 * r + 2; ++e) {
              sc[kg][i][e] = exp2_ftz(fmaf(sc[kg][i][e], scale_log2, -ref));
              sum += sc[kg][i][e];
            }
        l[r] = l[r] * alpha[r] + sum;
      }
      if (!first && __any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[0];
          o[i][2] *= alpha[1];
          o[i][3] *= alpha[1];
        }
      }
      first = false;
      if (ends && x.left > 0) fetch_q(x);  // lands while this unit ends
      // O += P V
      st = n % C::kHalf;
      if (!warp_wait(&full[st], (n / C::kHalf) & 1, abort_flag)) return false;
      base = smem_u32(sR) + st * C::kStage + vrow * 128;
#pragma unroll
      for (int kg = 0; kg < MT; ++kg) {
        const uint32_t p[4] = {pack2<BF16>(sc[kg][0][0], sc[kg][0][1]), pack2<BF16>(sc[kg][0][2], sc[kg][0][3]),
                               pack2<BF16>(sc[kg][1][0], sc[kg][1][1]), pack2<BF16>(sc[kg][1][2], sc[kg][1][3])};
        // keys past the sequence's end hold whatever was in the page: P is zero there, and
        // so must V be (0 * NaN is not).  A register has the keys 2 t and 2 t + 1 (+ 8).
        const int left = u.len - (key0 + slice * kKeysW + kg * 16 + 2 * t);
        const uint32_t keep0 = left >= 2 ? ~0u : left == 1 ? 0xffffu : 0u;
        const uint32_t keep1 = left >= 10 ? ~0u : left == 9 ? 0xffffu : 0u;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const int chunk = (i & 3) * 2 + (lane >> 4);
          uint32_t b[4];
          ldsm4_t(base + kg * 2048 + (i >> 2) * 8192 + ((chunk ^ (vrow & 7)) << 4), b);
          mma16816<BF16>(o[2 * i], p, b[0] & keep0, b[1] & keep1);
          mma16816<BF16>(o[2 * i + 1], p, b[2] & keep0, b[3] & keep1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      ++n;
    }
    // join the slices: [4 warps][16 rows][HD] fp32, columns in pairs, pair p of row g at
    // p ^ (g << 2) so that a warp's stores meet no bank twice.  The parts of the unit
    // before have been read when every warp has said so at its end.
    if (units > 0 && !warp_wait(&joined[0], (units - 1) & 1, abort_flag)) return false;
    float* part = reinterpret_cast<float*>(sQ);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float2* dst = reinterpret_cast<float2*>(part + (warp * 16 + g + 8 * r) * HD);
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) dst[(i * 4 + t) ^ (g << 2)] = make_float2(o[i][2 * r], o[i][2 * r + 1]);
      float sum = l[r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) s_ml[warp * 16 + g + 8 * r] = make_float2(m[r] - shift, sum);  // no token: -inf, 0
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&joined[1]);
    if (!warp_wait(&joined[1], units & 1, abort_flag)) return false;
    ++units;
    constexpr int V = HD / 32;
    const bool direct = whole && !cut_front;
    // rows warp, warp + 4, ..  Not unrolled: code that a unit runs once costs more in
    // issue than in latency (3 rows side by side: 4,000 cycles, so: 2,200)
#pragma unroll 1
    for (int pr = warp; pr < u.rows; pr += 4) {
      const int r = pr & 15, first = (pr >> 4) * kSlices;
      float2 ml[kSlices];
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kSlices; ++i) {
        ml[i] = s_ml[(first + i) * 16 + r];
        top = fmaxf(top, ml[i].x);
      }
      float acc[V] = {}, sum = 0.f;
#pragma unroll
      for (int i = 0; i < kSlices; ++i) {
        const float f = ml[i].y == 0.f ? 0.f : exp2_ftz(ml[i].x - top);  // a sum of NaN stays
        const float* src = part + ((first + i) * 16 + r) * HD + (((lane * V / 2) ^ ((r & 7) << 2)) << 1);
        sum += f * ml[i].y;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(f, src[e], acc[e]);
      }
      const int h = __shfl_sync(0xffffffffu, hg, pr);
      if (direct) {
        write_row<HD, BF16>(a, __shfl_sync(0xffffffffu, tok, pr), head * group + (h < 0 ? ~h : h), acc, top, sum,
                            h >= 0);
      } else {
        const long long slot = piece_slot(kFew, share, !cut_front, pr);
        float* dst = w.few.o + slot * HD + lane * V;
#pragma unroll
        for (int e = 0; e < V; ++e) dst[e] = acc[e];
        if (lane == 0) w.few.ml[slot] = piece_ml(top, sum, h >= 0);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&joined[0]);
    return true;
  }
};

// 16 TMEM columns of a row, not waited for.
MOE_DEV void tmem_st16_start(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(kAttThreads, 1)
    kv_attend_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const KvView c, const KvAttend a, const KaPtrs w, const int group,
                     const float scale_log2) {
  using C = KaCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sR = sQ + 2 * C::kQ;  // the K / V ring
  uint64_t* bars = reinterpret_cast<uint64_t*>(sR + C::kStages * C::kStage);
  uint64_t* full = bars;                       // [kStages]
  uint64_t* empty = full + C::kStages;         // [kStages]
  uint64_t* half_full = empty + C::kStages;     // [2][kHalf] the rings of singles and few rows
  uint64_t* half_empty = half_full + C::kStages;  // [2][kHalf]
  uint64_t* s_full = half_empty + C::kStages;   // [stream][buffer] S of a tile done
  uint64_t* p_full = s_full + 4;               // [stream][buffer] P of a tile written
  uint64_t* o_done = s_full + 8;               // [stream][buffer] P V of a tile done
  uint64_t* joined = s_full + 12;              // [stream][2] 4 warps: parts read, parts written
  uint64_t* ring_free = s_full + 16;           // the MMAs have let all stages go
  uint64_t* mma_done = s_full + 17;
  uint64_t* q_full = s_full + 18;              // [stream] Q tile of a pair written
  uint64_t* q_free = s_full + 20;              // [stream] every S of a pair done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 22);
  static_assert((4 * C::kStages + 23) * 8 <= 768, "barriers");
  float2* s_ml = reinterpret_cast<float2*>(bars + 96);  // [2][4][16]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);
      mbar_init(&half_full[i], 1);
      mbar_init(&half_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&joined[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_free[i], 1);
    }
    mbar_init(ring_free, 1);
    mbar_init(mma_done, 2);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int cta = blockIdx.x;
  if (warp >= 8) {
  regs_fewer<kRegsOther>();
  if (warp == 8) {
    // ------------------------------------------------------------ K / V tiles of pairs
    KaCursor x;
    x.init(w, kPair, KaCursor::start(w, kPair, cta), c.heads);
    KaRing ring{c, tk, tv, a.layer, full, empty, smem_u32(sR), C::kStages, C::kStage, C::kLoads, abort_flag};
    KaPages pg;
    bool ok = true;
    while (ok && x.left > 0) ok = ring.put_unit(x, pg);
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) record_error(c.err, DEV_TIMEOUT_EMPTY);
    }
    // every copy must land before the CTA exits, and every MMA have read its stage before
    // the other kinds use it
    ring.drain(ok);
    if (ok && lane == 0) mbar_arrive(ring_free);
  }
  if (warp == 11) {
    // ------------------------------------------------------------ Q tiles of pairs
    // as soon as every S of the unit before is done: under its last softmax and epilogue
    KaCursor x;
    x.init(w, kPair, KaCursor::start(w, kPair, cta), c.heads);
    bool ok = true;
    for (int n = 0; ok && x.left > 0; ++n) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (ok && n > 0) ok = warp_wait(&q_free[s], (n - 1) & 1, abort_flag);
        if (ok) {
          fetch_q<HD>(a, x.u, x.head, group, s * kTile, smem_u32(sQ) + s * C::kQ);
          cp_async_wait();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[s]);
        }
      }
      x.skip(min(x.left, x.u.tiles - x.tile));
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) record_error(c.err, DEV_TIMEOUT_FULL);
    }
    __syncwarp();
  }
  if (warp == 8 || warp == 11) {
    // ------------------------------------------------------------ K / V tiles of singles, few rows
    // a ring and a producer warp for each of the two warpgroups
    const int r = warp == 11;
    KaCursor x, y;
    x.init(w, kSingle, KaCursor::start(w, kSingle, 2 * cta + r), c.heads);
    y.init(w, kFew, KaCursor::start(w, kFew, 2 * cta + r), c.heads);
    if (x.left > 0 || y.left > 0) {
      // the pairs may run for long: a limit of about two minutes
      bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(ring_free, 0, abort_flag, 128 * kWaitLimitCycles));
      KaRing ring{c, tk, tv, a.layer, half_full + r * C::kHalf, half_empty + r * C::kHalf,
                  smem_u32(sR) + r * C::kHalf * C::kStage, C::kHalf, C::kStage, C::kLoads, abort_flag};
      KaPages pg;
      while (ok && x.left > 0) ok = ring.put_unit(x, pg);
      while (ok && y.left > 0) {
        ok = ring.put(y.u, y.head, y.tile, pg, false) && ring.put(y.u, y.head, y.tile, pg, true);
        y.next();
      }
      if (!ok) {
        *abort_flag = 1;
        if (lane == 0) record_error(c.err, DEV_TIMEOUT_EMPTY);
      }
      ring.drain(false);
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------------------------------------ Q and MMAs of a stream
    const int s = warp - 9;
    constexpr uint32_t fmt = BF16 ? 1 : 0;
    constexpr uint32_t id_s = ka_idesc(fmt, kKeys, 0), id_o = ka_idesc(fmt, HD, 1);
    const bool lead = elect_one();
    const int leader = __ffs(__ballot_sync(0xffffffffu, lead)) - 1;
    const uint32_t t_s = uniform(tmem + s * kTile), t_o = t_s + kOCols;
    const uint32_t q_smem = smem_u32(sQ) + s * C::kQ;
    const uint64_t dq = sw128_desc(q_smem);
    const int4 start_pair = KaCursor::start(w, kPair, cta), start_single = KaCursor::start(w, kSingle, 2 * cta + s);
    bool ok = true;
    int ns = 0, np = 0, nq = 0;  // S tiles, P tiles, units so far
    // The units of a cursor from a ring.  One lane waits and issues: S two tiles ahead of
    // P V, P V of the unit's last two tiles apart, with rows of V past the sequence's end
    // cleared first (by the whole warp).  Q comes from warp 11 for pairs; singles, whose
    // streams do not wait for each other, fetch their own.
    auto units = [&](KaCursor x, bool own_q, uint64_t* fullb, uint64_t* emptyb, uint8_t* ring, int stages,
                     int extra_arrivals) {
      const uint64_t dk0 = sw128_desc(smem_u32(ring)), dv0 = nmajor_desc(smem_u32(ring));
      int st = 0;
      uint32_t ph = 0;
      auto let_go = [&](int at) {
        for (int i = 0; i < extra_arrivals; ++i) mbar_arrive(&emptyb[at]);
        tc_commit(&emptyb[at]);
      };
      auto pass = [&]() {
        if (++st == stages) {
          st = 0;
          ph ^= 1;
        }
      };
      auto product = [&](bool first) -> bool {  // O += P V
        const int buf = np & 1;
        if (!mbar_wait_bounded(&fullb[st], ph, abort_flag) ||
            !mbar_wait_bounded(&p_full[2 * s + buf], (np >> 1) & 1, abort_flag))
          return false;
        tc_fence_after();
        const uint64_t dv = dv0 + static_cast<uint32_t>(st * (C::kStage >> 4));
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          tc_mma_f16_ts(t_o, t_s + buf * kKeys + k * 8, dv + k * (2048 >> 4), id_o, first && k == 0 ? 0u : 1u);
        tc_commit(&o_done[2 * s + buf]);
        let_go(st);
        ++np;
        pass();
        return true;
      };
      while (ok && x.left > 0) {
        const int nt = min(x.left, x.u.tiles - x.tile);
        const int behind = max(nt - 2, 0);
        if (own_q) {
          if (ns > 0 && !warp_wait(&s_full[2 * s + ((ns - 1) & 1)], ((ns - 1) >> 1) & 1, abort_flag)) ok = false;
          fetch_q<HD>(a, x.u, x.head, group, 0, q_smem);
          cp_async_wait();
          fence_proxy_async_smem();
          __syncwarp();
        } else {
          if (!warp_wait(&q_full[s], nq & 1, abort_flag)) ok = false;
          ++nq;
        }
        if (lead) {
          for (int j = -2; ok && j < behind; ++j) {
            if (j >= 0) ok = product(j == 0);
            if (ok && j + 2 < nt) {
              const int buf = ns & 1;
              ok = mbar_wait_bounded(&fullb[st], ph, abort_flag);
              // the buffer holds P of two tiles before until its product is done: products of
              // different shapes are not promised to run in the order of their issue.  (Without
              // the wait 4096 new on 4096 cached tokens took 1.19 ms instead of 1.25.)
              if (ok && ns >= 2) ok = mbar_wait_bounded(&o_done[2 * s + buf], ((ns - 2) >> 1) & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
              const uint64_t dk = dk0 + static_cast<uint32_t>(st * (C::kStage >> 4));
#pragma unroll
              for (int k = 0; k < HD / 16; ++k)  // offsets in the descriptors' units of 16 bytes
                tc_mma_f16(t_s + buf * kKeys, dq + (((k >> 2) * 16384 + (k & 3) * 32) >> 4),
                           dk + (((k >> 2) * kKeys * 128 + (k & 3) * 32) >> 4), id_s, k > 0 ? 1u : 0u);
              tc_commit(&s_full[2 * s + buf]);
              if (j + 3 == nt && !own_q) tc_commit(&q_free[s]);
              let_go(st);
              ++ns;
              pass();
            }
          }
        }
        __syncwarp();
        // what the one lane counted
        ok = __shfl_sync(0xffffffffu, ok, leader);
        st = __shfl_sync(0xffffffffu, st, leader);
        ph = __shfl_sync(0xffffffffu, ph, leader);
        ns = __shfl_sync(0xffffffffu, ns, leader);
        np = __shfl_sync(0xffffffffu, np, leader);
        for (int j = behind; ok && j < nt; ++j) {
          // keys past the sequence's end hold whatever was in the page: their rows of V
          // are zeroed, since P is zero there but 0 * NaN is not
          const int valid = x.u.len - (x.tile + j) * kKeys;
          if (valid < kKeys) {
            if (!warp_wait(&fullb[st], ph, abort_flag)) {
              ok = false;
              break;
            }
            for (int kb = 0; kb < C::kLoads; ++kb)
              for (int o = max(valid, 0) * 128 + lane * 16; o < kKeys * 128; o += 512)
                *reinterpret_cast<uint4*>(ring + st * C::kStage + kb * kKeys * 128 + o) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lead) ok = product(j == 0);
          __syncwarp();
          ok = __shfl_sync(0xffffffffu, ok, leader);
          st = __shfl_sync(0xffffffffu, st, leader);
          ph = __shfl_sync(0xffffffffu, ph, leader);
          np = __shfl_sync(0xffffffffu, np, leader);
        }
        x.skip(nt);
      }
    };
    KaCursor x;
    x.init(w, kPair, start_pair, c.heads);
    units(x, false, full, empty, sR, C::kStages, 0);
    x.init(w, kSingle, start_single, c.heads);
    if (ok) units(x, true, half_full + s * C::kHalf, half_empty + s * C::kHalf, sR + s * C::kHalf * C::kStage, C::kHalf, 3);
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) record_error(c.err, DEV_TIMEOUT_FULL);
    }
    if (lead) tc_commit(mma_done);  // no MMA may still write TMEM when it is released
    mbar_wait_drain(mma_done, 0);
    __syncwarp();
  }
  } else {
    // ------------------------------------------------------------ softmax
    regs_more<kRegsSoftmax>();
    const int s = warp >> 2;           // stream
    const int quad = warp & 3;         // TMEM lanes 32 * quad ..
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + lanes + s * kTile;           // S, then P, of this stream
    const uint32_t t_o = tmem + lanes + kOCols + s * kTile;  // O
    // P is scaled by 2^shift: f16 keeps probabilities down to 2^-31 of the largest
    // (the reference maximum may lag by 2^8: 2^15 at most, below f16's 65504)
    constexpr float shift = BF16 ? 0.f : 7.f;
    __half* out16 = static_cast<__half*>(a.out);
    bool ok = true;
    int nt = 0;  // tiles of this stream so far
    const int4 st_pair = KaCursor::start(w, kPair, cta), st_single = KaCursor::start(w, kSingle, 2 * cta + s),
               st_few = KaCursor::start(w, kFew, 2 * cta + s);
#pragma unroll 1
    for (int kind = kPair; kind <= kSingle && ok; ++kind) {
      const int share = kind ? 2 * cta + s : cta;
      const int part = kind ? 0 : s;  // the unit's rows of this warpgroup: part * 128 ..
      KaCursor x;
      x.init(w, kind, kind ? st_single : st_pair, c.heads);
      if (x.left <= 0) continue;
      bool cut_front = x.tile > 0;  // the unit began in an earlier share
      while (x.left > 0 && ok) {
        const KaUnit u = x.u;
        const int head = x.head;
        const int pr = part * kTile + quad * 32 + lane;
        const bool valid = pr < u.rows;
        const bool any = part * kTile + quad * 32 < u.rows;  // a row in this warp
        const int packed = u.r0 + (valid ? pr : 0);
        const int tok = packed / group, hg = packed - tok * group;
        // tokens that the row sees: all up to its own position
        const int seen = valid ? max(min(u.base + tok + 1, u.len), 0) : 0;
        float m = -INFINITY, l = 0.f;
        bool first = true, whole = true;
        for (bool ends = false; !ends; first = false) {
          ends = x.ends_unit();
          const int key0 = x.tile * kKeys;
          if (ends) whole = x.tile + 1 == u.tiles;
          x.next();
          const int buf = nt & 1;
          const uint32_t t_sb = t_s + buf * kKeys;
          if (!warp_wait(&s_full[2 * s + buf], (nt >> 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (any) {
            float sc[kKeys];
            load_s(t_sb, sc);
            const int lim = seen - key0;
            if (__any_sync(0xffffffffu, lim < kKeys)) {
#pragma unroll
              for (int j = 0; j < kKeys; ++j)
                if (j >= lim) sc[j] = -INFINITY;
            }
            float mx[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) mx[j] = fmaxf(sc[j], fmaxf(sc[j + 8], sc[j + 16]));
#pragma unroll
            for (int j = 24; j < kKeys; j += 16)
#pragma unroll
              for (int k = 0; k < 8; ++k)
                mx[k] = j + 8 < kKeys ? fmaxf(mx[k], fmaxf(sc[j + k], sc[j + 8 + k])) : fmaxf(mx[k], sc[j + k]);
            const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                    fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * scale_log2;
            // m, the maximum that P, l and O refer to, moves (and l and O are rescaled)
            // only when it grows by more than 2^8
            const bool grow = valid && top - m > 8.f;
            float alpha = 1.f;
            if (grow) {
              alpha = exp2f(m - top);
              m = top;
            }
            if (!first && __any_sync(0xffffffffu, grow)) {
              // O must be complete up to the tile before (s_full says so up to two before)
              if (!warp_wait(&o_done[2 * s + (buf ^ 1)], ((nt - 1) >> 1) & 1, abort_flag)) {
                ok = false;
                break;
              }
              tc_fence_after();
#pragma unroll
              for (int i = 0; i < HD / 16; ++i) {
                float o[16];
                tmem_ld16(t_o + i * 16, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] *= alpha;
                tmem_st16(t_o + i * 16, o);
              }
            }
            // P in chunks of 32 keys: the conversions and TMEM stores of one run under the
            // exponentials of the next
            const float ref = m == -INFINITY ? 0.f : m - shift;
            const uint64_t scale2 = pair_of(scale_log2, scale_log2), nref2 = pair_of(-ref, -ref);
#pragma unroll
            for (int i = 0; i < kKeys / 32; ++i) {
              uint32_t pk[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float* e = sc + i * 32 + 2 * j;
                const float2 x2 = split_pair(fma_pair(pair_of(e[0], e[1]), scale2, nref2));
                e[0] = exp2_ftz(x2.x);
                e[1] = exp2_ftz(x2.y);
                pk[j] = pack2<BF16>(e[0], e[1]);
              }
              tmem_st16_start(t_sb + i * 16, pk);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * s + buf]);
            // the row sum, off the path to the product with V
            uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kKeys / 2; ++j) sum[j & 3] = add_pair(sum[j & 3], pair_of(sc[2 * j], sc[2 * j + 1]));
            const float2 sum2 = split_pair(add_pair(add_pair(sum[0], sum[1]), add_pair(sum[2], sum[3])));
            l = l * alpha + (sum2.x + sum2.y);
          } else {
            tc_fence_before();
            if (lane == 0) mbar_arrive(&p_full[2 * s + buf]);
          }
          ++nt;
        }
        if (!ok) break;
        if (!warp_wait(&o_done[2 * s + ((nt - 1) & 1)], ((nt - 1) >> 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (any) {
          if (whole && !cut_front) {
            const long long row = static_cast<long long>(u.row0) + tok;
            const int h = head * group + hg;
            const bool saw = seen > 0;  // as in write_row
            const float inv = 1.f / l;
            // a thread writes its own row: its 32 lanes meet 32 lines in every store, so
            // the stores are as wide as they can be
            __half* dst = out16 + row * a.os[0] + h * a.os[1];
            const bool wide = !((reinterpret_cast<uintptr_t>(out16) | (a.os[0] * 2) | (a.os[1] * 2)) & 31);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
              float o[32];
              tmem_ld32(t_o + i * 32, o);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                uint32_t pk[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  pk[j] = saw ? pack2<BF16>(o[k * 16 + 2 * j] * inv, o[k * 16 + 2 * j + 1] * inv) : 0u;
                if (valid && wide) {
                  store32(dst + i * 32 + k * 16, pk);
                } else if (valid) {
                  uint4* d4 = reinterpret_cast<uint4*>(dst + i * 32 + k * 16);
                  d4[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                  d4[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
                }
              }
            }
            if (valid && a.lse)
              a.lse[row * a.ls[0] + h * a.ls[1]] =
                  saw ? (m - shift + log2f(l)) * 0.6931471805599453f : -INFINITY;
          } else {
            // a piece: unnormalised, to the share's slot 0 (its first unit) or 1 (its last)
            const KaList l_k = w.kind(kind);
            const long long slot = piece_slot(kind, share, !cut_front, pr);
            float* dst = l_k.o + slot * HD;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
              float o[32];
              tmem_ld32(t_o + i * 32, o);
              if (valid) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  uint32_t v[8];
#pragma unroll
                  for (int j = 0; j < 8; ++j) v[j] = __float_as_uint(o[k * 8 + j]);
                  store32(dst + i * 32 + k * 8, v);
                }
              }
            }
            if (valid) l_k.ml[slot] = piece_ml(m - shift, l, seen > 0);
          }
        }
        tc_fence_before();  // O is read: the next unit's first product may overwrite it
        cut_front = false;
      }
    }
    // few rows: this warpgroup's share
    if (ok) {
      KaFew<HD, BF16> f{c, a, w, group, scale_log2, sQ + s * C::kQ, sR + s * C::kHalf * C::kStage,
                        half_full + s * C::kHalf, half_empty + s * C::kHalf, joined + 2 * s, s_ml + s * 64,
                        abort_flag};
      f.n = 2 * st_single.w;  // the ring has gone round for the singles
      const int share = 2 * cta + s;
      KaCursor x;
      x.init(w, kFew, st_few, c.heads);
      if (x.left > 0) f.fetch_q(x);
      while (ok && x.left > 0) {
        const int rows = x.u.rows;
        ok = rows <= 16 ? f.template unit<1>(x, share) : f.template unit<2>(x, share);
      }
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) record_error(c.err, DEV_TIMEOUT_TMEM_FULL);
    }
  }
  pdl_release();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ merge
// Joins the pieces of cut units, in share order: 16 rows a CTA and step, two rows a warp.
// A kernel of its own, since its reading (two or more fp32 pieces a row) wants the whole
// GPU: joined by the last warp of a unit inside the attention kernel, 33 mixed chunks took
// 293 us instead of 241 (at that time).
template <int HD, bool BF16>
__global__ void __launch_bounds__(256) kv_merge_kernel(const KvAttend a, const KaPtrs w, const int group) {
  pdl_enter();
  constexpr int V = HD / 32, P = 4;  // pieces at a time, for loads in flight
  const int lane = threadIdx.x & 31;
  const int r0 = blockIdx.y * kMergeRows + 2 * (threadIdx.x >> 5);
  const int n = *w.n_merge;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int4 e = *reinterpret_cast<const int4*>(w.merge + i);
    const int item = w.merge[i].item;
    const int kind = e.x, first = e.y, last = e.z;
    const KaList l = w.kind(kind);
    const int4 u0 = *reinterpret_cast<const int4*>(l.list + item);  // seq, row0, r0, rows
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, acc[2][V] = {};
    for (int base = first; base <= last; base += 32) {
      // shares of the unit that have tiles
      const int mine = base + lane;
      const bool has = mine <= last && l.start[mine].count > 0;
      if (r0 >= u0.w) break;
      for (uint32_t todo = __ballot_sync(0xffffffffu, has); todo;) {
        float2 ml[P][2];
        float v[P][2][V];
        bool on[P];
#pragma unroll
        for (int q = 0; q < P; ++q) {
          on[q] = todo != 0;
          const int s = base + (on[q] ? __ffs(todo) - 1 : 0);
          todo &= todo - 1;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const long long slot = piece_slot(kind, s, s == first, min(r0 + j, u0.w - 1));
            ml[q][j] = l.ml[slot];
            const float* src = l.o + slot * HD + lane * V;
            if constexpr (V == 4) {
              const float4 t = *reinterpret_cast<const float4*>(src);
              v[q][j][0] = t.x; v[q][j][1] = t.y; v[q][j][2] = t.z; v[q][j][3] = t.w;
            } else {
              const float2 t = *reinterpret_cast<const float2*>(src);
              v[q][j][0] = t.x; v[q][j][1] = t.y;
            }
          }
        }
        // the running maximum moves with the pieces, in share order
#pragma unroll
        for (int q = 0; q < P; ++q) {
          if (!on[q]) break;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // a piece without a visible token (sum 0) holds nothing, whatever its rows say; a
            // sum of NaN counts, with or without a maximum
            const bool some = ml[q][j].y != 0.f;
            const float up = fmaxf(top[j], ml[q][j].x);
            const float keep = top[j] == -INFINITY ? 0.f : exp2_ftz(top[j] - up);
            const float f = some ? exp2_ftz(ml[q][j].x - up) : 0.f;
            top[j] = up;
            sum[j] = sum[j] * keep + (some ? f * ml[q][j].y : 0.f);
#pragma unroll
            for (int x = 0; x < V; ++x) acc[j][x] = acc[j][x] * keep + (some ? f * v[q][j][x] : 0.f);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int packed = u0.z + r0 + j, tok = packed / group;
      if (r0 + j < u0.w)
        write_row<HD, BF16>(a, static_cast<long long>(u0.y) + tok, e.w * group + packed - tok * group, acc[j], top[j],
                            sum[j], top[j] != -INFINITY);
    }
  }
}

template <int HD, bool BF16>
static cudaError_t ka_launch(const KvView& c, const CUtensorMap& tk, const CUtensorMap& tv,
                             const KvBatch& b, const KvAttend& a, char* ws, int num_sms, cudaStream_t s) {
  const int group = a.heads / c.heads;
  const KaWs l = ka_ws(c, a.heads, b.rows, b.n, num_sms);
  KaPtrs w{};
  for (int k = 0; k < kKinds; ++k) {
    KaList& d = k == kPair ? w.pair : k == kSingle ? w.single : w.few;
    d.start = reinterpret_cast<KaStart*>(ws + l.start[k]);
    d.list = reinterpret_cast<KaUnit*>(ws + l.list[k]);
    d.pre = reinterpret_cast<long long*>(ws + l.pre[k]);
    d.o = reinterpret_cast<float*>(ws + l.o[k]);
    d.ml = reinterpret_cast<float2*>(ws + l.ml[k]);
  }
  w.merge = reinterpret_cast<KaMerge*>(ws + l.merge);
  w.n_merge = reinterpret_cast<int*>(ws + l.n_merge);
  constexpr size_t smem = KaCfg<HD>::kSmem;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    const cudaError_t st = cudaFuncSetAttribute(kv_attend_kernel<HD, BF16>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                static_cast<int>(smem));
    if (st != cudaSuccess) return st;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  MOE_PDL(kv_plan_kernel, dim3(1), dim3(kPlanT), 0, s, c, b, group, num_sms, w, l.cap[0]);
  MOE_PDL(kv_attend_kernel<HD, BF16>, dim3(num_sms), dim3(kAttThreads), smem, s, tk, tv, c, a, w, group,
          static_cast<float>(a.scale * 1.4426950408889634));
  const int64_t most = std::min<int64_t>(static_cast<int64_t>(b.rows) * group, 2 * kTile);
  MOE_PDL(kv_merge_kernel<HD, BF16>, dim3(num_sms, static_cast<int>((most + kMergeRows - 1) / kMergeRows)),
          dim3(256), 0, s, a, w, group);
  return cudaSuccess;
}

cudaError_t kv_launch_attend(const KvView& c, const CUtensorMap& tk, const CUtensorMap& tv, bool bf16,
                             const KvBatch& b, const KvAttend& a, void* ws, int num_sms, cudaStream_t s) {
  char* p = static_cast<char*>(ws);
  if (c.hd == 128)
    return bf16 ? ka_launch<128, true>(c, tk, tv, b, a, p, num_sms, s)
                : ka_launch<128, false>(c, tk, tv, b, a, p, num_sms, s);
  return bf16 ? ka_launch<64, true>(c, tk, tv, b, a, p, num_sms, s)
              : ka_launch<64, false>(c, tk, tv, b, a, p, num_sms, s);
}

}  // namespace moe
