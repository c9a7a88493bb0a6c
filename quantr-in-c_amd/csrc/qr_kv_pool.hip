// qr_kv_pool.hip -- a KV pool that sequences share: its page operations, the
// 8-bit store and load of a ragged batch's rows, and their C entry points
// (qr_kv_pool_* of qr_hip.h; the attention's kernels are in qr_kv_attn.hip).
// No counterpart in the reference, whose cache holds one sequence
// (src/model.c:82-88, src/runtime.c:74-92).
//
// The state of a pool (tables, lengths, reference counts) lives on the device
// and every call is a fixed sequence of launches that wait for nothing, so a
// serving step can be captured whole.  Nothing depends on the order of
// atomics: they only count.
#include <math.h>

#include "qr_kv_pool.h"
#include "qr_lanes.h"

namespace qr {
namespace {

constexpr int kPlan = 1024;  // threads of the planning workgroup

// Exclusive prefix sums of one value per thread of a kPlan-thread workgroup;
// *total receives the sum.  tmp: 17 values of LDS.
__device__ inline long block_scan(long v, long* tmp, long* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  long s = v;
  for (int d = 1; d < 64; d <<= 1) {
    const long o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 63) tmp[w] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    long a = 0;
    for (int i = 0; i < kPlan / 64; i++) {
      const long t = tmp[i];
      tmp[i] = a;
      a += t;
    }
    tmp[16] = a;
  }
  __syncthreads();
  *total = tmp[16];
  return tmp[w] + s - v;
}

// Four reference counts from page i on (behind the last page: `pad`).
__device__ inline int4 refs4(const int32_t* refs, int i, int n, int pad) {
  int4 r;
  r.x = i < n ? refs[i] : pad;
  r.y = i + 1 < n ? refs[i + 1] : pad;
  r.z = i + 2 < n ? refs[i + 2] : pad;
  r.w = i + 3 < n ? refs[i + 3] : pad;
  return r;
}

struct PageState {
  int32_t *table, *len, *refs;
  int n_pages, n_seqs, max_pages, page_shift;
};

__device__ inline int pages_of(long tokens, int shift) {
  return (int)((tokens + ((1l << shift) - 1)) >> shift);
}

// The pages of a copy-on-write or a compaction, as the copying launch reads them.
struct CopyPlan {
  int32_t* count;
  int32_t *src, *dst;
};

// ---- extend -----------------------------------------------------------------
// One workgroup plans: which listed sequences copy their last page, how many
// pages each takes (prefix sums), the free pages in order, and then writes the
// tables.  It is bound by the latency of its few dependent loads, so what does
// not depend on others (the list, the first 4096 reference counts) is loaded at once,
// and what is needed again stays in registers and LDS; a larger grid would have to
// agree on the plan first.
constexpr int kFirst = 4 * kPlan;   // pages whose reference counts are held in LDS
constexpr int kFreeLds = 1536;      // free pages listed in LDS; more in scratch memory
__global__ __launch_bounds__(kPlan) void k_pages_extend(PageState p, const int32_t* seqs,
                                                        const int32_t* add, int n, CopyPlan plan,
                                                        int32_t* freelist, int32_t* status) {
  __shared__ long tmp[17];
  __shared__ int bad;
  __shared__ uint32_t seen[QR_KV_MAX_SEQS / 32];
  __shared__ int32_t last[QR_KV_MAX_LIST];   // the partly filled last page, -1: none
  __shared__ uint32_t off[QR_KV_MAX_LIST];   // first slot among the pages taken
  __shared__ __align__(16) int32_t first[kFirst];  // reference counts
  __shared__ int32_t freed[kFreeLds];
  constexpr int kEach = QR_KV_MAX_LIST / kPlan;
  const int tid = threadIdx.x;
  int s[kEach], more[kEach], len[kEach];
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int i = tid + j * kPlan;
    s[j] = i < n ? seqs[i] : 0;
    more[j] = i < n ? add[i] : 0;
  }
  const int4 head = refs4(p.refs, 4 * tid, p.n_pages, 1);
  for (int i = tid; i < (p.n_seqs + 31) / 32; i += kPlan) seen[i] = 0;
  if (tid == 0) bad = 0;
  *reinterpret_cast<int4*>(&first[4 * tid]) = head;
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const bool ok = (unsigned)s[j] < (unsigned)p.n_seqs;
    len[j] = ok ? p.len[s[j]] : -1;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int i = tid + j * kPlan;
    if (i >= n) continue;
    int l = -1;
    const long L = len[j];
    if (L < 0 || more[j] < 0 || L + more[j] > ((long)p.max_pages << p.page_shift)) {
      bad = 1;
    } else {
      if (atomicOr(&seen[s[j] >> 5], 1u << (s[j] & 31)) & (1u << (s[j] & 31))) bad = 1;
      if (more[j] > 0 && (L & ((1l << p.page_shift) - 1))) {
        l = p.table[(size_t)s[j] * p.max_pages + (L >> p.page_shift)];
        if ((unsigned)l >= (unsigned)p.n_pages) bad = 1;
      }
    }
    last[i] = l;
  }
  __syncthreads();
  if (bad) {
    if (tid == 0) {
      plan.count[0] = 0;
      if (status) status[0] = QR_ERR_INVALID;
    }
    return;
  }
  // Of the listed sequences that share a last page, the earlier ones copy
  // while others still hold it.
  long base = 0, copies = 0;
  int cow[kEach];
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    cow[j] = 0;
    if (j * kPlan >= n) continue;  // the whole workgroup
    const int i = tid + j * kPlan;
    long need = 0;
    if (i < n) {
      const int l = last[i];
      if (l >= 0) {
        const int r = l < kFirst ? first[l] : p.refs[l];
        if (r > 1) {
          int before = 0;
          for (int k = 0; k < i; k++) before += last[k] == l;
          cow[j] = before < r - 1;
        }
      }
      need = cow[j] + pages_of((long)len[j] + more[j], p.page_shift) -
             pages_of(len[j], p.page_shift);
    }
    long tot;
    const long ex = block_scan((need << 16) + cow[j], tmp, &tot);
    if (i < n) {
      off[i] = (uint32_t)(base + (ex >> 16));
      if (cow[j]) {
        const long k = copies + (ex & 0xFFFF);
        plan.src[k] = last[i];
        plan.dst[k] = (int32_t)off[i];  // the slot, until the page is known
      }
    }
    base += tot >> 16;
    copies += tot & 0xFFFF;
  }
  // the free pages in ascending order, as many as are taken
  int32_t* const list = base <= kFreeLds ? freed : freelist;
  long found = 0;
  for (int i0 = 0; i0 < p.n_pages && found < base; i0 += 4 * kPlan) {
    const int i = i0 + 4 * tid;
    const int4 r = i0 == 0 ? head : refs4(p.refs, i, p.n_pages, 1);
    const int f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
    long tot;
    long k = found + block_scan(f[0] + f[1] + f[2] + f[3], tmp, &tot);
    for (int j = 0; j < 4; j++)
      if (f[j]) {
        if (k < base) list[k] = i + j;
        k++;
      }
    found += tot;
  }
  __syncthreads();
  if (found < base) {
    if (tid == 0) {
      plan.count[0] = 0;
      if (status) status[0] = QR_ERR_NOMEM;
    }
    return;
  }
  // each sequence's first page by its own thread, further ones by all
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int i = tid + j * kPlan;
    if (i >= n) continue;
    p.len[s[j]] = len[j] + more[j];
    const long end = i + 1 < n ? (long)off[i + 1] : base;
    if ((long)off[i] >= end) continue;
    const int page = list[off[i]];
    p.table[(size_t)s[j] * p.max_pages + pages_of(len[j], p.page_shift) - cow[j]] = page;
    p.refs[page] = 1;
    if (cow[j]) atomicAdd(&p.refs[last[i]], -1);
    last[i] = pages_of(len[j], p.page_shift) - cow[j];  // where its pages begin
  }
  __syncthreads();
  for (long k = tid; k < base; k += kPlan) {
    int lo = 0, hi = n - 1;  // the last sequence whose first slot is not behind k
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long)off[mid] <= k)
        lo = mid;
      else
        hi = mid - 1;
    }
    if ((long)off[lo] == k) continue;
    const int page = list[k];
    p.table[(size_t)seqs[lo] * p.max_pages + last[lo] + (int)(k - off[lo])] = page;
    p.refs[page] = 1;
  }
  for (long k = tid; k < copies; k += kPlan) plan.dst[k] = list[plan.dst[k]];
  if (tid == 0) {
    plan.count[0] = (int32_t)copies;
    if (status) status[0] = QR_OK;
  }
}

// ---- compact ------------------------------------------------------------------
// One workgroup: L = the pages in use, then the free pages below L and the
// used ones from L on, each in order: as many of one as of the other.
__global__ __launch_bounds__(kPlan) void k_pages_plan(PageState p, CopyPlan plan, int32_t* to,
                                                      int32_t* n_live) {
  __shared__ long tmp[17];
  const int tid = threadIdx.x;
  long mine = 0, live;
  for (int i = 4 * tid; i < p.n_pages; i += 4 * kPlan) {
    const int4 r = refs4(p.refs, i, p.n_pages, 0);
    mine += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0);
  }
  block_scan(mine, tmp, &live);
  long holes = 0, movers = 0;
  for (int i0 = 0; i0 < p.n_pages; i0 += 4 * kPlan) {
    const int i = i0 + 4 * tid;
    const int4 r = refs4(p.refs, i, p.n_pages, 0);
    const int u[4] = {r.x > 0, r.y > 0, r.z > 0, r.w > 0};
    long h = 0, m = 0;
    for (int j = 0; j < 4; j++) {
      if (i + j < live)
        h += !u[j];
      else
        m += u[j];
    }
    long tot;
    const long ex = block_scan((h << 32) + m, tmp, &tot);
    h = holes + (ex >> 32);
    m = movers + (ex & 0xFFFFFFFFl);
    for (int j = 0; j < 4 && i + j < p.n_pages; j++) {
      if (i + j < live) {
        if (!u[j]) plan.dst[h++] = i + j;
      } else if (u[j]) {
        plan.src[m++] = i + j;
      }
      to[i + j] = u[j] ? i + j : -1;
    }
    holes += tot >> 32;
    movers += tot & 0xFFFFFFFFl;
  }
  __syncthreads();
  for (long k = tid; k < movers; k += kPlan) to[plan.src[k]] = plan.dst[k];
  if (tid == 0) {
    plan.count[0] = (int32_t)movers;
    if (n_live) n_live[0] = (int32_t)live;
  }
}

// The planned pages of all layers, 16 KiB of a page's values (and with its first
// piece the page's scales) by a workgroup at a time: bound by HBM.  With
// `to` (a compaction), tables and reference counts follow.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kCopyPiece = 16 * 1024;
__global__ __launch_bounds__(256) void k_pages_copy(PageState p, int8_t* data, float* scale,
                                                    long page_bytes, int page_scales, int n_layers,
                                                    CopyPlan plan, const int32_t* to) {
  const int count = plan.count[0];
  const int pieces = (int)((page_bytes + kCopyPiece - 1) / kCopyPiece);
  const long total = (long)count * n_layers * pieces;
  for (long w = blockIdx.x; w < total; w += gridDim.x) {
    const int piece = (int)(w % pieces);
    const long pl = w / pieces;
    const int layer = (int)(pl % n_layers);
    const int k = (int)(pl / n_layers);
    const long src = (long)layer * p.n_pages + plan.src[k];
    const long dst = (long)layer * p.n_pages + plan.dst[k];
    const long b0 = (long)piece * kCopyPiece;
    const int n16 = (int)((page_bytes - b0 < kCopyPiece ? page_bytes - b0 : kCopyPiece) / 16);
    const u32x4* s = reinterpret_cast<const u32x4*>(data + src * page_bytes + b0);
    u32x4* d = reinterpret_cast<u32x4*>(data + dst * page_bytes + b0);
    if (n16 == kCopyPiece / 16) {
      u32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = s[threadIdx.x + 256 * j];
#pragma unroll
      for (int j = 0; j < 4; j++) d[threadIdx.x + 256 * j] = v[j];
    } else {
      for (int i = threadIdx.x; i < n16; i += 256) d[i] = s[i];
    }
    if (piece == 0) {
      const float2* ss = reinterpret_cast<const float2*>(scale + src * page_scales);
      float2* sd = reinterpret_cast<float2*>(scale + dst * page_scales);
      for (int i = threadIdx.x; i < page_scales / 2; i += 256) sd[i] = ss[i];
    }
  }
  if (!to) return;
  const long entries = (long)p.n_seqs * p.max_pages;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < entries; i += (long)gridDim.x * 256) {
    const int g = p.table[i];
    if (g >= 0) p.table[i] = g < p.n_pages ? to[g] : -1;
  }
  for (long k = (long)blockIdx.x * 256 + threadIdx.x; k < count; k += (long)gridDim.x * 256) {
    p.refs[plan.dst[k]] = p.refs[plan.src[k]];
    p.refs[plan.src[k]] = 0;
  }
}

// ---- assign -------------------------------------------------------------------
// Every workgroup checks the list; then each takes whole columns of the table:
// it reads the listed rows' entries of a column, and only then writes them, so
// a sequence may be a source and a destination at once.
__global__ __launch_bounds__(kPlan) void k_pages_assign(PageState p, const int32_t* dst,
                                                        const int32_t* src, int n, int cols,
                                                        int32_t* status) {
  __shared__ int bad;
  __shared__ uint32_t seen[QR_KV_MAX_SEQS / 32];
  const int tid = threadIdx.x;
  for (int i = tid; i < (p.n_seqs + 31) / 32; i += kPlan) seen[i] = 0;
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kPlan) {
    const int d = dst[i], s = src[i];
    if ((unsigned)d >= (unsigned)p.n_seqs || (unsigned)s >= (unsigned)p.n_seqs)
      bad = 1;
    else if (atomicOr(&seen[d >> 5], 1u << (d & 31)) & (1u << (d & 31)))
      bad = 1;
  }
  __syncthreads();
  if (bad) {
    if (blockIdx.x == 0 && tid == 0 && status) status[0] = QR_ERR_INVALID;
    return;
  }
  // cols columns at a time, n * cols <= QR_KV_MAX_LIST entries
  constexpr int kEach = QR_KV_MAX_LIST / kPlan;
  for (int c0 = blockIdx.x * cols; n > 0 && c0 < p.max_pages; c0 += gridDim.x * cols) {
    int was[kEach], now[kEach];
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      const int e = tid + j * kPlan, c = c0 + e / n;
      was[j] = now[j] = -1;
      if (e < n * cols && c < p.max_pages) {
        was[j] = p.table[(size_t)dst[e % n] * p.max_pages + c];
        now[j] = p.table[(size_t)src[e % n] * p.max_pages + c];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      const int e = tid + j * kPlan, c = c0 + e / n;
      if (e < n * cols && c < p.max_pages && was[j] != now[j]) {
        p.table[(size_t)dst[e % n] * p.max_pages + c] = now[j];
        if ((unsigned)was[j] < (unsigned)p.n_pages) atomicAdd(&p.refs[was[j]], -1);
        if ((unsigned)now[j] < (unsigned)p.n_pages) atomicAdd(&p.refs[now[j]], 1);
      }
    }
  }
  if (blockIdx.x != 0) return;
  int l[kEach];
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int i = tid + j * kPlan;
    l[j] = i < n ? p.len[src[i]] : 0;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int i = tid + j * kPlan;
    if (i < n) p.len[dst[i]] = l[j];
  }
  if (tid == 0 && status) status[0] = QR_OK;
}

// ---- trim, reset ----------------------------------------------------------------
__global__ __launch_bounds__(256) void k_pages_trim(PageState p, const int32_t* seqs,
                                                    const int32_t* keep, int n, int32_t* status) {
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256)
    if ((unsigned)seqs[i] >= (unsigned)p.n_seqs || keep[i] < 0) bad = 1;
  __syncthreads();
  if (status && blockIdx.x == 0 && threadIdx.x == 0) status[0] = bad ? QR_ERR_INVALID : QR_OK;
  if (bad) return;
  const long total = (long)n * p.max_pages;
  for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
    const int i = (int)(e / p.max_pages), c = (int)(e % p.max_pages);
    const int s = seqs[i];
    if (c >= pages_of(keep[i], p.page_shift) && p.table[(size_t)s * p.max_pages + c] != -1) {
      // exchanged, so that a sequence listed twice gives each page back once
      const int g = atomicExch(&p.table[(size_t)s * p.max_pages + c], -1);
      if ((unsigned)g < (unsigned)p.n_pages) atomicAdd(&p.refs[g], -1);
    }
    if (c == 0) atomicMin(&p.len[s], keep[i]);
  }
}

__global__ __launch_bounds__(256) void k_pages_reset(PageState p) {
  const long entries = (long)p.n_seqs * p.max_pages;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < entries; i += (long)gridDim.x * 256) {
    p.table[i] = -1;
    if (i < p.n_seqs) p.len[i] = 0;
  }
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.n_pages; i += (long)gridDim.x * 256)
    p.refs[i] = 0;
}

// ---- store, load ----------------------------------------------------------------
// What a wave needs of its slot: the block, the tokens of it that rows stand
// for, and the sequence's rows.
struct BlockRows {
  SeqRows s;
  int piece;     // of the sequence's slots, < 0: none
  bool any;      // the block holds rows
  bool there;    // and its page exists
  size_t blk;    // index of the block in the layer
  int first;     // token of the block that row row0 stands for (may be < 0)
};

// Slots of a sequence: one for each block that its rows touch, of which m rows
// touch at most floor(end / 16) - floor(start / 16) + 2.
__device__ inline BlockRows block_rows(const PoolView& p, const Ragged& r, int slot, int kvh) {
  BlockRows b;
  b.any = b.there = false;
  b.s = slot_rows(p, r, slot, kKvBlock, 2, &b.piece);
  b.s.len = seq_len(p, b.s);
  if (b.piece < 0 || b.s.m == 0) return b;
  const int pos0 = b.s.len - b.s.m;  // of the first row; < 0 where there are more rows than tokens
  const long lb = (long)(pos0 < 0 ? 0 : pos0) / kKvBlock + b.piece;
  if (lb * kKvBlock >= b.s.len) return b;
  b.any = true;
  b.first = pos0 - (int)lb * kKvBlock;
  const int page = page_at(p, b.s.seq, (int)((lb << 4) >> p.page_shift));
  if (page < 0) return b;
  b.there = true;
  b.blk = block_at(p, page, kvh, (int)lb & ((1 << (p.page_shift - 4)) - 1));
  return b;
}

// A block's scale, and what its values and its older scale are multiplied by (a power of two)
// so that nothing below under- or overflows.
struct Step {
  float s, inv, mul, was;
};
__device__ inline Step step_of(float s, float was) {
  Step k;
  k.mul = s < 0x1p-100f ? 0x1p100f : s > 0x1p100f ? 0x1p-100f : 1.0f;
  k.s = s * k.mul;
  k.was = was * k.mul;
  k.inv = 1.0f / k.s;
  return k;
}

// x / s rounded to the nearest even integer, for |x| <= 127 s but for rounding.  The
// product with 1 / s is within one integer of it, and what it leaves of x is a multiple of the
// smaller of both ulps below 2^24 of them, so the fused multiply-add forms it
// exactly and decides.
__device__ inline int quantized(float x, const Step& k) {
  const float y = x * k.mul;
  float q = rintf(y * k.inv);
  const float rem = __builtin_fmaf(-q, k.s, y), two = 2.0f * fabsf(rem);
  const bool odd = ((int)q & 1) != 0;
  q += (two > k.s) | ((two == k.s) & odd) ? copysignf(1.0f, rem) : 0.0f;
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  if (!(fabsf(x) <= 3.402823466e+38f)) q = x != x ? 0.0f : copysignf(127.0f, x);
  return k.s > 0.0f ? (int)q : 0;
}

// An older value under a grown scale, rounded the same way.  Its product with the old scale
// is p + e exactly; where the rest r of p is near half a step, 2 r - s is exact, and the sign of
// its sum with 2 e decides.
__device__ inline int requantized(int q, const Step& k) {
  const float a = fabsf((float)q), p = a * k.was, e = __builtin_fmaf(a, k.was, -p);
  float m = rintf(p * k.inv);
  const float r = __builtin_fmaf(-m, k.s, p);
  const float over = __builtin_fmaf(2.0f, fabsf(r), -k.s) + copysignf(2.0f, r) * e;
  const bool odd = ((int)m & 1) != 0;
  m += (over > 0.0f) | ((over == 0.0f) & odd) ? copysignf(1.0f, r) : 0.0f;
  return q < 0 ? -(int)m : (int)m;
}

// A wave per (block, kv head, K or V): its new rows in registers, the largest
// of them, the scale, then the 8-bit values beside what the block holds.  K in
// quads of columns (4 * HD of them in all), V a column of 16 tokens per
// lane: both store what a lane has in one piece.  HBM bounds many rows,
// latency few.
template <int HD>
__global__ __launch_bounds__(256) void k_pool_store(PoolView p, Ragged r, const float* k,
                                                    const float* v, long stride, int slots) {
  const int lane = threadIdx.x & 63;
  const int w = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int side = w & 1, slot = w >> 1, kvh = blockIdx.y;
  if (slot >= slots) return;
  const BlockRows b = block_rows(p, r, slot, kvh);
  if (!b.there) return;
  const float* x = (side ? v : k) + (size_t)kvh * HD;
  float* sc = p.scale + 2 * b.blk + side;
  int8_t* out = p.data + b.blk * (2 * kKvBlock * HD) + side * kKvBlock * HD;
  const bool held = b.first > 0;
  const float was = held ? *sc : 0.0f;
  auto fresh = [&](int t) { return t >= b.first && t - b.first < b.s.m; };
  auto row = [&](int t) { return x + (size_t)(b.s.row0 + t - b.first) * stride; };
  float amax = 0.0f;
  auto take = [&](float f) {
    const float a = fabsf(f);
    if (a <= 3.402823466e+38f) amax = fmaxf(amax, a);
  };
  auto scale_of = [&]() {
    const float s = fmaxf(was, wave_max(amax) / 127.0f);
    if (lane == 0) *sc = s;
    return s;
  };
  if (side == 0) {
    constexpr int Q = HD / 4, N = (kKvBlock * Q + 63) / 64;
    float4 f[N];
    int old[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int e = lane + 64 * j, t = e / Q;
      f[j] = make_float4(0, 0, 0, 0);
      old[j] = 0;
      if (e < kKvBlock * Q && fresh(t)) f[j] = *reinterpret_cast<const float4*>(row(t) + e % Q * 4);
      if (e < kKvBlock * Q && t < b.first) old[j] = reinterpret_cast<const int*>(out)[e];
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      take(f[j].x);
      take(f[j].y);
      take(f[j].z);
      take(f[j].w);
    }
    const float s = scale_of();
    const Step st = step_of(s, was);
    const bool grew = held && s > was;
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int e = lane + 64 * j;
      const int a = quantized(f[j].x, st), c = quantized(f[j].y, st), d = quantized(f[j].z, st),
                g = quantized(f[j].w, st);
      if (e < kKvBlock * Q && fresh(e / Q))
        reinterpret_cast<int*>(out)[e] = (a & 255) | (c & 255) << 8 | (d & 255) << 16 | g << 24;
    }
    if (grew) {
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int e = lane + 64 * j, u = old[j];
        const int a = requantized((int8_t)u, st), c = requantized((int8_t)(u >> 8), st),
                  d = requantized((int8_t)(u >> 16), st), g = requantized(u >> 24, st);
        if (e < kKvBlock * Q && e / Q < b.first)
          reinterpret_cast<int*>(out)[e] = (a & 255) | (c & 255) << 8 | (d & 255) << 16 | g << 24;
      }
    }
  } else {
    constexpr int N = (HD + 63) / 64;
    float f[N][kKvBlock];
    int4 old[N];
    const bool all = b.first <= 0 && b.s.m + b.first >= kKvBlock;
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = lane + 64 * j;
      old[j] = make_int4(0, 0, 0, 0);
      if (!all && c < HD) old[j] = *reinterpret_cast<const int4*>(out + c * kKvBlock);
    }
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int t = 0; t < kKvBlock; t++) {
        const int c = lane + 64 * j;
        f[j][t] = c < HD && fresh(t) ? row(t)[c] : 0.0f;
      }
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int t = 0; t < kKvBlock; t++) take(f[j][t]);
    const float s = scale_of();
    const Step st = step_of(s, was);
    const bool grew = held && s > was;
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = lane + 64 * j;
      int u[4] = {old[j].x, old[j].y, old[j].z, old[j].w};
      auto put = [&](int t, int q) {
        u[t >> 2] = (u[t >> 2] & ~(255 << 8 * (t & 3))) | (q & 255) << 8 * (t & 3);
      };
      if (grew) {
#pragma unroll
        for (int t = 0; t < kKvBlock; t++)
          if (t < b.first) put(t, requantized((int8_t)(u[t >> 2] >> 8 * (t & 3)), st));
      }
#pragma unroll
      for (int t = 0; t < kKvBlock; t++)
        if (fresh(t)) put(t, quantized(f[j][t], st));
      if (c < HD) *reinterpret_cast<int4*>(out + c * kKvBlock) = make_int4(u[0], u[1], u[2], u[3]);
    }
  }
}

// The same split backwards.  A slot without a page reads the layer's first
// block, which is there, and takes zeros for it (with a branch around the loads a store and
// load of 64 x 1 tokens took 13.1 us for 11.0).
template <int HD>
__global__ __launch_bounds__(256) void k_pool_load(PoolView p, Ragged r, float* k, float* v,
                                                   long stride, int slots) {
  const int lane = threadIdx.x & 63;
  const int w = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int side = w & 1, slot = w >> 1, kvh = blockIdx.y;
  if (slot >= slots) return;
  float* x = (side ? v : k) + (size_t)kvh * HD;
  const BlockRows b = block_rows(p, r, slot, kvh);
  if (b.piece < 0) return;
  // Of the sequence's rows, 16 for each of its slots: those before position 0.
  const int none = b.s.m - b.s.len;
  for (int t = kKvBlock * b.piece; t < none && t < kKvBlock * (b.piece + 1); t++)
    for (int c = lane; c < HD; c += 64) x[(size_t)(b.s.row0 + t) * stride + c] = 0.0f;
  if (!b.any) return;
  const float s = b.there ? p.scale[2 * b.blk + side] : 0.0f;
  const int there = b.there ? -1 : 0;
  const int8_t* in = p.data + (b.there ? b.blk : 0) * (2 * kKvBlock * HD) + side * kKvBlock * HD;
  auto fresh = [&](int t) { return t >= b.first && t - b.first < b.s.m; };
  auto row = [&](int t) { return x + (size_t)(b.s.row0 + t - b.first) * stride; };
  if (side == 0) {
    constexpr int Q = HD / 4, N = (kKvBlock * Q + 63) / 64;
    int block[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int e = lane + 64 * j;
      block[j] = e < kKvBlock * Q ? reinterpret_cast<const int*>(in)[e] : 0;
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int e = lane + 64 * j, t = e / Q, u = block[j] & there;
      if (e >= kKvBlock * Q || !fresh(t)) continue;
      *reinterpret_cast<float4*>(row(t) + e % Q * 4) =
          make_float4((float)(int8_t)u * s, (float)(int8_t)(u >> 8) * s,
                      (float)(int8_t)(u >> 16) * s, (float)(u >> 24) * s);
    }
  } else {
    constexpr int N = (HD + 63) / 64;
    int4 block[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = lane + 64 * j;
      block[j] = make_int4(0, 0, 0, 0);
      if (c < HD) block[j] = *reinterpret_cast<const int4*>(in + c * kKvBlock);
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = lane + 64 * j, u[4] = {block[j].x & there, block[j].y & there, block[j].z & there,
                                               block[j].w & there};
#pragma unroll
      for (int t = 0; t < kKvBlock; t++)
        if (c < HD && fresh(t)) row(t)[c] = (float)(int8_t)(u[t >> 2] >> 8 * (t & 3)) * s;
    }
  }
}

// ---- host ---------------------------------------------------------------------
int pool_check(const qr_ctx* c, const qr_kv_pool* p, const char* who) {
  if (!c) return set_error(QR_ERR_INVALID, "%s: null ctx", who);
  if (!p) return set_error(QR_ERR_INVALID, "%s: null pool", who);
  if (p->n_layers <= 0 || p->n_pages <= 0 || p->n_kv_heads <= 0 || p->n_kv_heads > 1024 ||
      p->max_pages <= 0 ||
      p->n_seqs <= 0 || p->n_seqs > QR_KV_MAX_SEQS)
    return set_error(QR_ERR_INVALID, "%s: pool of %d layers, %d pages, %d kv heads, %d x %d table",
                     who, p->n_layers, p->n_pages, p->n_kv_heads, p->n_seqs, p->max_pages);
  if (p->page < kKvBlock || p->page > 65536 || (p->page & (p->page - 1)))
    return set_error(QR_ERR_INVALID, "%s: page %d (a power of two, 16 to 65536)", who, p->page);
  if (p->head_dim <= 0 || p->head_dim % 32 || p->head_dim > 256)
    return set_error(QR_ERR_INVALID, "%s: head_dim %d (a multiple of 32, <= 256)", who, p->head_dim);
  if ((long)p->max_pages * p->page > 1l << 30)
    return set_error(QR_ERR_INVALID, "%s: %d pages of %d tokens exceed 2^30", who, p->max_pages,
                     p->page);
  if ((long)p->n_pages * p->n_kv_heads * (p->page / kKvBlock) > 1l << 31)
    return set_error(QR_ERR_INVALID, "%s: more than 2^31 blocks a layer", who);
  if (!p->data || !p->scale || !p->table || !p->len || !p->refs)
    return set_error(QR_ERR_INVALID, "%s: null pointer in the pool", who);
  if (((uintptr_t)p->data & 15) || ((uintptr_t)p->scale & 7) || ((uintptr_t)p->table & 3) ||
      ((uintptr_t)p->len & 3) || ((uintptr_t)p->refs & 3))
    return set_error(QR_ERR_INVALID, "%s: pool alignment (data 16 bytes, scale 8)", who);
  return QR_OK;
}

PageState page_state(const qr_kv_pool* p) {
  PageState s;
  s.table = p->table;
  s.len = p->len;
  s.refs = p->refs;
  s.n_pages = p->n_pages;
  s.n_seqs = p->n_seqs;
  s.max_pages = p->max_pages;
  s.page_shift = __builtin_ctz((unsigned)p->page);
  return s;
}

long page_bytes(const qr_kv_pool* p) {
  return (long)p->n_kv_heads * (p->page / kKvBlock) * 2 * kKvBlock * p->head_dim;
}
int page_scales(const qr_kv_pool* p) { return p->n_kv_heads * (p->page / kKvBlock) * 2; }

PoolView layer_view(const qr_kv_pool* p, int layer) {
  PoolView v;
  v.data = p->data + (long)layer * p->n_pages * page_bytes(p);
  v.scale = p->scale + (long)layer * p->n_pages * page_scales(p);
  v.table = p->table;
  v.len = p->len;
  v.n_pages = p->n_pages;
  v.n_kv_heads = p->n_kv_heads;
  v.hd = p->head_dim;
  v.n_seqs = p->n_seqs;
  v.max_pages = p->max_pages;
  v.page_shift = __builtin_ctz((unsigned)p->page);
  return v;
}

int list_check(const void* a, const void* b, int n, const char* who) {
  if (n < 0 || n > QR_KV_MAX_LIST)
    return set_error(QR_ERR_INVALID, "%s: a list of %d (0..%d)", who, n, QR_KV_MAX_LIST);
  if (n > 0 && (!a || !b)) return set_error(QR_ERR_INVALID, "%s: null list", who);
  return QR_OK;
}

#define KV_HIP(call, what)                                                                \
  do {                                                                                    \
    hipError_t e_ = (call);                                                               \
    if (e_ != hipSuccess) return set_error(QR_ERR_HIP, "%s: %s", what, hipGetErrorString(e_)); \
  } while (0)

// The planned copies: as many workgroups as the most pages that may move need,
// at most eight per CU (each then takes several pieces).
hipError_t copy_launch(const qr_kv_pool* p, long most, CopyPlan plan, const int32_t* to,
                       hipStream_t st) {
  const long pieces = (page_bytes(p) + kCopyPiece - 1) / kCopyPiece;
  long grid = most * p->n_layers * pieces;
  if (grid > 2048) grid = 2048;
  if (grid < 1) grid = 1;
  hipLaunchKernelGGL(k_pages_copy, dim3((unsigned)grid), dim3(256), 0, st, page_state(p), p->data,
                     p->scale, page_bytes(p), page_scales(p), p->n_layers, plan, to);
  return hipGetLastError();
}

int ragged_check(const qr_kv_pool* p, int layer, const int32_t* start, int n, int T,
                 const char* who) {
  if (layer < 0 || layer >= p->n_layers)
    return set_error(QR_ERR_INVALID, "%s: layer %d of %d", who, layer, p->n_layers);
  if (n < 0 || n > QR_KV_MAX_SEQS || T < 0 || T > QR_KV_MAX_ROWS)
    return set_error(QR_ERR_INVALID, "%s: %d sequences, %d rows", who, n, T);
  if (n > 0 && T > 0 && !start) return set_error(QR_ERR_INVALID, "%s: null start", who);
  return QR_OK;
}

int rows_check(const void* k, const void* v, long stride, long width, const char* who) {
  if (!k || !v) return set_error(QR_ERR_INVALID, "%s: null rows", who);
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15) || (stride & 3) || stride < width)
    return set_error(QR_ERR_INVALID,
                     "%s: rows must be 16-byte aligned, their stride (%ld) a multiple of 4, >= %ld",
                     who, stride, width);
  return QR_OK;
}

#define KV_HD_SWITCH(hd, F)   \
  switch (hd) {               \
    case 32: F(32); break;    \
    case 64: F(64); break;    \
    case 96: F(96); break;    \
    case 128: F(128); break;  \
    case 160: F(160); break;  \
    case 192: F(192); break;  \
    case 224: F(224); break;  \
    default: F(256); break;   \
  }

}  // namespace
}  // namespace qr

using namespace qr;

extern "C" {

int qr_kv_pool_reset(qr_ctx* c, const qr_kv_pool* p) {
  const char* who = "qr_kv_pool_reset";
  const int rc = pool_check(c, p, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  long grid = ((long)p->n_seqs * p->max_pages + p->n_pages + 255) / 256;
  if (grid > 1024) grid = 1024;
  hipLaunchKernelGGL(k_pages_reset, dim3((unsigned)grid), dim3(256), 0, ctx_stream(c),
                     page_state(p));
  KV_HIP(hipGetLastError(), "k_pages_reset");
  return QR_OK;
}

int qr_kv_pool_extend(qr_ctx* c, const qr_kv_pool* p, const int32_t* seqs, const int32_t* add,
                      int n, int32_t* status) {
  const char* who = "qr_kv_pool_extend";
  int rc = pool_check(c, p, who);
  if (!rc) rc = list_check(seqs, add, n, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  void* w = nullptr;
  rc = ctx_scratch_get(c, ((size_t)p->n_pages + 2 * QR_KV_MAX_LIST + 4) * 4, who, &w);
  if (rc) return rc;
  CopyPlan plan;
  plan.count = static_cast<int32_t*>(w);
  plan.src = plan.count + 4;
  plan.dst = plan.src + QR_KV_MAX_LIST;
  hipLaunchKernelGGL(k_pages_extend, dim3(1), dim3(kPlan), 0, ctx_stream(c), page_state(p), seqs,
                     add, n, plan, plan.dst + QR_KV_MAX_LIST, status);
  KV_HIP(hipGetLastError(), "k_pages_extend");
  if (n > 0) KV_HIP(copy_launch(p, n, plan, nullptr, ctx_stream(c)), "k_pages_copy");
  return QR_OK;
}

int qr_kv_pool_assign(qr_ctx* c, const qr_kv_pool* p, const int32_t* dst, const int32_t* src,
                      int n, int32_t* status) {
  const char* who = "qr_kv_pool_assign";
  int rc = pool_check(c, p, who);
  if (!rc) rc = list_check(dst, src, n, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  const int cols = n > 0 ? QR_KV_MAX_LIST / n : 1;
  int grid = n > 0 ? (p->max_pages + cols - 1) / cols : 1;
  if (grid > 512) grid = 512;
  hipLaunchKernelGGL(k_pages_assign, dim3(grid), dim3(kPlan), 0, ctx_stream(c), page_state(p), dst,
                     src, n, cols, status);
  KV_HIP(hipGetLastError(), "k_pages_assign");
  return QR_OK;
}

int qr_kv_pool_trim(qr_ctx* c, const qr_kv_pool* p, const int32_t* seqs, const int32_t* keep,
                    int n, int32_t* status) {
  const char* who = "qr_kv_pool_trim";
  int rc = pool_check(c, p, who);
  if (!rc) rc = list_check(seqs, keep, n, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  long grid = ((long)n * p->max_pages + 255) / 256;
  if (grid > 1024) grid = 1024;
  if (grid < 1) grid = 1;
  hipLaunchKernelGGL(k_pages_trim, dim3((unsigned)grid), dim3(256), 0, ctx_stream(c),
                     page_state(p), seqs, keep, n, status);
  KV_HIP(hipGetLastError(), "k_pages_trim");
  return QR_OK;
}

int qr_kv_pool_compact(qr_ctx* c, const qr_kv_pool* p, int32_t* map, int32_t* n_live) {
  const char* who = "qr_kv_pool_compact";
  int rc = pool_check(c, p, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  void* w = nullptr;
  rc = ctx_scratch_get(c, (3 * (size_t)p->n_pages + 4) * 4, who, &w);
  if (rc) return rc;
  CopyPlan plan;
  plan.count = static_cast<int32_t*>(w);
  plan.src = plan.count + 4;
  plan.dst = plan.src + p->n_pages;
  int32_t* to = map ? map : plan.dst + p->n_pages;
  hipLaunchKernelGGL(k_pages_plan, dim3(1), dim3(kPlan), 0, ctx_stream(c), page_state(p), plan, to,
                     n_live);
  KV_HIP(hipGetLastError(), "k_pages_plan");
  KV_HIP(copy_launch(p, (p->n_pages + 1) / 2, plan, to, ctx_stream(c)), "k_pages_copy");
  return QR_OK;
}

int qr_kv_pool_store(qr_ctx* c, const qr_kv_pool* p, int layer, const int32_t* seqs,
                     const int32_t* start, int n, int T, const float* k, const float* v,
                     long stride) {
  const char* who = "qr_kv_pool_store";
  int rc = pool_check(c, p, who);
  if (!rc) rc = ragged_check(p, layer, start, n, T, who);
  if (rc) return rc;
  if (n == 0 || T == 0) return QR_OK;
  rc = rows_check(k, v, stride, (long)p->n_kv_heads * p->head_dim, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  const Ragged r{seqs, start, n, T};
  const int slots = T / kKvBlock + 2 * n;
#define KV_STORE(HD)                                                                             \
  hipLaunchKernelGGL(k_pool_store<HD>, dim3((slots + 1) / 2, p->n_kv_heads), dim3(256), 0,          \
                     ctx_stream(c), layer_view(p, layer), r, k, v, stride, slots)
  KV_HD_SWITCH(p->head_dim, KV_STORE);
#undef KV_STORE
  KV_HIP(hipGetLastError(), "k_pool_store");
  return QR_OK;
}

int qr_kv_pool_load(qr_ctx* c, const qr_kv_pool* p, int layer, const int32_t* seqs,
                    const int32_t* start, int n, int T, float* k, float* v, long stride) {
  const char* who = "qr_kv_pool_load";
  int rc = pool_check(c, p, who);
  if (!rc) rc = ragged_check(p, layer, start, n, T, who);
  if (rc) return rc;
  if (n == 0 || T == 0) return QR_OK;
  rc = rows_check(k, v, stride, (long)p->n_kv_heads * p->head_dim, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  const Ragged r{seqs, start, n, T};
  const PoolView view = layer_view(p, layer);
  const int slots = T / kKvBlock + 2 * n;
#define KV_LOAD(HD)                                                                              \
  hipLaunchKernelGGL(k_pool_load<HD>, dim3((slots + 1) / 2, p->n_kv_heads), dim3(256), 0,           \
                     ctx_stream(c), view, r, k, v, stride, slots)
  KV_HD_SWITCH(p->head_dim, KV_LOAD);
#undef KV_LOAD
  KV_HIP(hipGetLastError(), "k_pool_load");
  return QR_OK;
}

int qr_kv_pool_attention(qr_ctx* c, const qr_kv_pool* p, int layer, const int32_t* seqs,
                         const int32_t* start, int n, int T, int n_heads, const float* q,
                         long q_stride, float* out, long out_stride, int max_len, int window,
                         float scale) {
  const char* who = "qr_kv_pool_attention";
  int rc = pool_check(c, p, who);
  if (!rc) rc = ragged_check(p, layer, start, n, T, who);
  if (rc) return rc;
  if (n_heads <= 0 || n_heads > 16384 || n_heads % p->n_kv_heads)
    return set_error(QR_ERR_INVALID, "%s: heads %d / kv heads %d", who, n_heads, p->n_kv_heads);
  if (max_len < 0 || window < 0 || !(scale <= 3.402823466e+38f))
    return set_error(QR_ERR_INVALID, "%s: max_len %d, window %d, scale %g", who, max_len, window,
                     (double)scale);
  if (n == 0 || T == 0) return QR_OK;
  rc = rows_check(q, out, q_stride, (long)n_heads * p->head_dim, who);
  if (!rc) rc = rows_check(q, out, out_stride, (long)n_heads * p->head_dim, who);
  if (rc) return rc;
  KV_HIP(hipSetDevice(ctx_device(c)), "hipSetDevice");
  const Ragged r{seqs, start, n, T};
  const PoolView view = layer_view(p, layer);
  const int cap = p->max_pages * p->page;
  if (max_len == 0 || max_len > cap) max_len = cap;
  if (window >= cap) window = 0;  // no sequence is longer
  void* w = nullptr;
  const size_t need = kv_attention_scratch(view, r, n_heads, max_len, window);
  if (need) {
    rc = ctx_scratch_get(c, need, who, &w);
    if (rc) return rc;
  }
  KV_HIP(kv_attention_launch(view, r, n_heads, q, q_stride, out, out_stride, max_len, window,
                             scale > 0.0f ? scale : 1.0f / sqrtf((float)p->head_dim), w,
                             ctx_stream(c)),
         "k_pool_attn");
  return QR_OK;
}

}  // extern "C"
