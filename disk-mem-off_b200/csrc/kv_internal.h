// Paged K/V cache: the view that its kernels take, and the launchers shared by
// kv_pages.cu (pages, append) and kv_attend.cu (attention over the cache).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "moe_internal.h"

namespace moe {

// Everything a cache kernel needs, by value.  Strides are in bytes: layer, page,
// head, row (a row is one token's head_dim values, contiguous).
struct KvView {
  char* k;
  char* v;
  int64_t ks[4], vs[4];
  int layers, pages, heads, page, page_shift, hd;
  int* table;  // [nseq][max_blocks]
  int nseq, max_blocks;
  int* len;    // [nseq]
  int* refs;   // [pages]
  // scratch (kv_scratch_words)
  int* err;
  int* count;  // pages to copy, written by the kernel that plans a copy
  int* ok;     // a batch may be written (kv_check_kernel)
  int* src;    // [cap] pages to copy from
  int* dst;    // [cap] pages to copy to
  int* rows;   // [cap] rows of each page to copy
  int* list;   // [pages] free pages / new page of each page
  int* off;    // [nseq] first free page of each entry
};

// The caller's scratch, zeroed once: 16 words (error word, copy count, batch check), then
// the arrays above.
inline size_t kv_scratch_words(int pages, int nseq) {
  const size_t cap = static_cast<size_t>(pages > nseq ? pages : nseq);
  return 16 + 3 * cap + static_cast<size_t>(pages) + nseq;
}

// Most sequences of a cache: a bitmap of them is checked in shared memory.
constexpr int kKvMaxSeqs = 65536;
// Most SMs that a cache's kernels are spread over (a B200 has 148): the attention's plan
// keeps a number for each share in shared memory.
constexpr int kKvMaxSms = 192;

// One batch of new rows: row r of entry e is q_start[e] <= r < q_start[e + 1].
struct KvBatch {
  const int* seqs;     // [n]
  const int* q_start;  // [n + 1]
  int n;
  int rows;  // rows of the tensors; those from q_start[n] on are left alone
};

inline size_t bitmap_bytes(const KvView& v) { return static_cast<size_t>((v.nseq + 31) / 32) * 4; }

#ifdef __CUDACC__
// Whether rows may be written for a batch, for every thread of the CTA: offsets that begin
// at 0 or later, do not decrease and end within the rows, and no sequence with rows in two
// entries (both would write its last places).  What is wrong is recorded.  bits:
// bitmap_bytes of shared memory; U: entries of a thread at a time, for loads in flight.
template <int U>
MOE_DEV bool check_batch(const KvView& c, const KvBatch& b, uint32_t* bits) {
  for (int i = threadIdx.x; i < (c.nseq + 31) / 32; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int i0 = threadIdx.x; i0 < b.n; i0 += U * blockDim.x) {
    int at[U], end[U], s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * blockDim.x;
      at[u] = end[u] = s[u] = 0;
      if (i < b.n) {
        at[u] = b.q_start[i];
        end[u] = b.q_start[i + 1];
        s[u] = b.seqs[i];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] < 0 || end[u] < at[u] || end[u] > b.rows) {
        record_error(c.err, DEV_BAD_LENGTH);
        bad = true;
      } else if (end[u] > at[u] && s[u] >= 0 && s[u] < c.nseq &&
                 (atomicOr(&bits[s[u] >> 5], 1u << (s[u] & 31)) >> (s[u] & 31) & 1u)) {
        record_error(c.err, DEV_BAD_SEQ);
        bad = true;
      }
    }
  }
  return !__syncthreads_or(bad);
}
// Every CTA of a writing kernel knows before it writes: up to kCheckHere entries it checks
// the batch itself, of more kv_check_kernel has left the answer in *c.ok.  Append of n rows
// of n sequences, without a check / checked in each CTA / by the kernel: 64: 2.7 / 3.0 us,
// 512: 3.1 / 4.2, 1,024: 4.0 / 7.4 / 6.5, 4,096: 5.6 / 24.7 / 9.8, 16,384: 19 / 170 / 30.
constexpr int kCheckHere = 512;
MOE_DEV bool batch_ok(const KvView& c, const KvBatch& b, uint32_t* bits) {
  return b.n <= kCheckHere ? check_batch<1>(c, b, bits) : *c.ok != 0;
}

// The entry of row r: the last e with q_start[e] <= r, -1 before the first (n > 0), by a
// warp (32 probes a round, one round at least: a single entry may begin after row r too).
MOE_DEV int entry_of_row(const int* __restrict__ q_start, int n, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;  // answer in [lo, hi), once q_start[lo] <= r
  do {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool le = at < hi && q_start[at] <= r;
    const uint32_t m = __ballot_sync(0xffffffffu, le);
    if (!m) return -1;
    const int j = 31 - __clz(m);
    hi = min(hi, lo + (j + 1) * step);
    lo += j * step;
  } while (hi - lo > 1);
  return lo;
}
#endif

// Before a kernel that calls batch_ok.
cudaError_t kv_launch_check(const KvView& c, const KvBatch& b, cudaStream_t s);
cudaError_t kv_launch_append(const KvView& c, const KvBatch& b, int layer, const void* k,
                             const void* v, const int64_t (&ks)[2], const int64_t (&vs)[2],
                             int num_sms, cudaStream_t s);

struct KvAttend {
  const void* q;
  void* out;
  float* lse;         // null: not wanted
  int64_t qs[2], os[2], ls[2];  // token and head strides in elements
  int heads;
  int layer;
  float scale;
};
size_t kv_attend_workspace(const KvView& c, int heads, int rows, int n_seqs, int num_sms);
cudaError_t kv_launch_attend(const KvView& c, const CUtensorMap& tk, const CUtensorMap& tv,
                             bool bf16, const KvBatch& b, const KvAttend& a, void* ws,
                             int num_sms, cudaStream_t s);

bool make_tmap_pool(CUtensorMap* map, const void* base, bool bf16, const KvView& c,
                    const int64_t (&strides)[4], std::string* err);

}  // namespace moe

// The opaque handle of the C ABI: host memory only.
struct MoeKvCache {
  moe::KvView v;
  CUtensorMap tk, tv;
  bool bf16;
  int device;
  int num_sms;
};
