// qr_logprobs.hip -- log probabilities of given tokens, entropy and the best
// alternatives of rows of logits (qr_logprobs of qr_hip.h), in one pass.
//
// With m = max x, S = sum e^(x - m) and U = sum e^(x - m) (x - m):
//   log p_t = (x_t - m) - log S,   -sum p log p = log S - U / S.
// A lane keeps its own m, S and U and lifts them when its maximum grows (S e^d,
// (U + S d) e^d with d the maximum's step down), so the row is read once, nothing
// is exchanged on the way, and the sums are 32-bit sums of few terms each.  The
// best tokens come from the same read: a wave keeps up to 64 of its best as 64-bit
// keys (the logit's order, then the lower index), one a lane, and
// looks at a segment of 1024 logits only where one of them beats the n-th.
// Long rows are bound by HBM; few rows are cut into parts that a second launch
// joins, bound by latency.
#include <math.h>

#include "qr_internal.h"
#include "qr_lanes.h"

namespace qr {
namespace {

constexpr int kSeg = 1024;   // logits of a wave's step: 16 a lane
constexpr int kLpWaves = 4;
constexpr int kBuf = 512;    // keys of a wave's buffer
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.44269504088896340736f;
// Below this a difference's exponential is 0 in fp32; it stands for -inf, whose
// product with 0 would be NaN.
constexpr float kFar = -200.0f;
constexpr int kFew = 4;          // parts that one wave joins
constexpr int kMaxLists = 1024;  // parts of a row
constexpr int kChoose = 4096;    // keys that one of its waves chooses from: 64 lists
static_assert(kChoose >= 64 * QR_LOGPROBS_MAX_TOP, "the lists that hold the best tokens");

typedef unsigned long long u64;
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LogprobArgs {
  const float* x;
  long stride;
  int rows, vocab;
  const int32_t* targets;
  float *lp, *entropy;
  int32_t* rank;
  int n_top;
  int32_t* top_id;
  float* top_lp;
  int splits, chunk;   // parts of a row, logits of each (a multiple of kSeg)
  u64* keys;           // [row][part][64]
  float* stats;        // [row][part][4]: m, S, U, and the logits ahead of the target
};

// A lane's or a row's sums.  S is NaN where one of the logits is NaN or +inf.
struct Sums {
  float m, S, U;
  int ahead;   // logits ahead of the target's
};

__device__ inline float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

__device__ inline Sums join(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - r.m, kFar), db = fmaxf(b.m - r.m, kFar);
  const float fa = exp_of(da), fb = exp_of(db);
  r.S = a.S * fa + b.S * fb;
  r.U = (a.U + a.S * da) * fa + (b.U + b.S * db) * fb;
  r.ahead = a.ahead + b.ahead;
  return r;
}

__device__ inline Sums wave_join(Sums s) {
  const float m = wave_max(s.m), d = fmaxf(s.m - m, kFar), e = exp_of(d);
  s.U = wave_sum((s.U + s.S * d) * e);
  s.S = wave_sum(s.S * e);
  s.m = m;
  int a = s.ahead;
  a += (int)lane_xor<1>((uint32_t)a);
  a += (int)lane_xor<2>((uint32_t)a);
  a += (int)lane_xor<7>((uint32_t)a);
  a += (int)lane_xor<15>((uint32_t)a);
  a += (int)lane_xor<16>((uint32_t)a);
  a += (int)lane_xor<32>((uint32_t)a);
  s.ahead = a;
  return s;
}

// Order-preserving 32 bits of a logit that is no NaN; -0 equals 0.  Never 0.
__device__ inline uint32_t order_of(float x) {
  const int b = __builtin_bit_cast(int, x + 0.0f);
  return (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// One compare-exchange of a descending network with the lane that differs by X:
// the lane without X's highest bit keeps the larger.
template <int X>
__device__ inline void exchange(u64& k) {
  constexpr int kTop = X >= 32 ? 32 : X >= 16 ? 16 : X >= 8 ? 8 : X >= 4 ? 4 : X >= 2 ? 2 : 1;
  const u64 o = lane_xor_64<X>(k);
  k = ((threadIdx.x & kTop) == 0) == (o > k) ? o : k;
}
__device__ inline void halves16(u64& k) {
  exchange<8>(k);
  exchange<4>(k);
  exchange<2>(k);
  exchange<1>(k);
}
// 64 keys, descending over the lanes (a network whose merges begin mirrored; by way of LDS it
// takes half as long again).
__device__ inline u64 sort64(u64 k) {
  exchange<1>(k);
  exchange<3>(k);
  exchange<1>(k);
  exchange<7>(k);
  exchange<2>(k);
  exchange<1>(k);
  exchange<15>(k);
  exchange<4>(k);
  exchange<2>(k);
  exchange<1>(k);
  exchange<31>(k);
  halves16(k);
  exchange<63>(k);
  exchange<16>(k);
  halves16(k);
  return k;
}
// The 64 largest of two descending lists, descending.
__device__ inline u64 merge64(u64 a, u64 b) {
  const u64 r = lane_xor_64<63>(b);
  u64 k = r > a ? r : a;
  exchange<32>(k);
  exchange<16>(k);
  halves16(k);
  return k;
}
__device__ inline u64 largest64(u64 k) {
  u64 o;
#define STEP(X) \
  o = lane_xor_64<X>(k); \
  k = o > k ? o : k;
  STEP(1) STEP(2) STEP(7) STEP(15) STEP(16) STEP(32)
#undef STEP
  return k;
}

// A wave's best logits: `key` one a lane, descending, 0 where there are fewer, and
// `count` more in its buffer.  At least n of the logits seen are of order `bound` or
// above (0: fewer seen), so a later one must be above it to be among the best n.
struct Best {
  u64 key;
  int count;
  uint32_t bound;
  float value;   // of the bound; -inf without one
  bool sorted;   // the buffer has been sorted into the list before
};

// The buffer into the list.
__device__ inline void best_flush(Best& b, int n, const u64* buf) {
  const int lane = threadIdx.x & 63;
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (int i = 0; i < b.count; i += 64)
    b.key = merge64(b.key, sort64(i + lane < b.count ? buf[i + lane] : 0));
  __builtin_amdgcn_wave_barrier();
  b.count = 0;
  b.sorted = true;
  const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)(b.key >> 32), n - 1);
  b.bound = o > b.bound ? o : b.bound;
}

// A segment's logits that may be among the best join the buffer, which is sorted into
// the list (and the bound raised) once it holds 64: a row in no order brings a few of
// them a segment, and sorting each time took most of a long row's time (512 x 151936 logits,
// 20 best: 97 us).  o: the logits' orders (0: no logit), at(j): their places.  With more than 64
// of them, those below the n-th largest of the lanes' maxima cannot be among the best
// n and are left out first; it is found bit by bit to 16 bits, whose rounding down lets a
// few more in.
template <class At>
__device__ inline void best_add(Best& b, uint32_t (&o)[16], int n, u64* buf, At at) {
  const int lane = threadIdx.x & 63;
  uint32_t mx = 0;
  int c = 0;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    c += __popcll(__ballot(o[j] > b.bound));
    mx = o[j] > mx ? o[j] : mx;
  }
  uint32_t least = b.bound + 1;
  if (c > 64) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; bit--) {
      const uint32_t u = t | 1u << bit;
      if (__popcll(__ballot(mx >= u)) >= n) t = u;
    }
    if (t > least) {
      least = t;
      b.bound = t;
    }
  }
#pragma unroll 1
  for (int q = 0; q < 4; q++) {
    if (b.count > kBuf - 256) best_flush(b, n, buf);  // many equal logits
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const u64 v = __ballot(o[j] >= least);
      if (o[j] >= least)
        buf[b.count + __popcll(v & ((1ull << lane) - 1))] =
            (u64)o[j] << 32 | (uint32_t)~at(4 * q + j);
      b.count += __popcll(v);
    }
#pragma unroll
    for (int j = 0; j < 12; j++) o[j] = o[j + 4];
  }
  if (b.count >= 64) best_flush(b, n, buf);
  b.value = b.bound ? value_of(b.bound) : kNegInf;
}

// Of c keys in LDS (held in R registers a lane, c <= 64 R, or read again each time, R = 0),
// those that can be among the best n, one a lane in no order, by one wave: a bound that at
// least n of them reach is raised bit by bit until 64 or fewer are left.  Where it ends with
// more (equal logits), the 64 best in order.
template <int R>
__device__ inline u64 choose(u64* cand, int c, int n) {
  const int lane = threadIdx.x & 63;
  uint32_t t = 0;
  int count = c;
  if (c > 64) {
    uint32_t o[R > 0 ? R : 1];
#pragma unroll
    for (int j = 0; j < R; j++)
      o[j] = 64 * j + lane < c ? (uint32_t)(cand[64 * j + lane] >> 32) : 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0 && count > 64; bit--) {
      const uint32_t u = t | 1u << bit;
      int m = 0;
#pragma unroll
      for (int j = 0; j < R; j++) m += __popcll(__ballot(o[j] >= u));
      if (R == 0)
        for (int i = lane; i - lane < c; i += 64)
          m += __popcll(__ballot(i < c && (uint32_t)(cand[i] >> 32) >= u));
      if (m >= n) {
        t = u;
        count = m;
      }
    }
    // to the front, in place: a key never moves behind where it is read
    count = 0;
#pragma unroll 1
    for (int i = 0; i < c; i += 64) {
      const u64 k = i + lane < c ? cand[i + lane] : 0;
      const bool in = k != 0 && (uint32_t)(k >> 32) >= t;
      const u64 v = __ballot(in);
      if (in) cand[count + __popcll(v & ((1ull << lane) - 1))] = k;
      count += __popcll(v);
      __builtin_amdgcn_wave_barrier();
    }
  }
  u64 key = lane < count ? cand[lane] : 0;
  if (count > 64) {
    key = sort64(key);
#pragma unroll 1
    for (int i = 64; i < count; i += 64)
      key = merge64(key, sort64(i + lane < count ? cand[i + lane] : 0));
  }
  return key;
}

// The row's results, by one wave with the whole row's sums and sorted list; ok: the row
// has a target, whose logit is xt.
__device__ inline void finish(const LogprobArgs& a, int r, const Sums& s, u64 key, bool ok,
                              float xt) {
  const int lane = threadIdx.x & 63;
  const bool bad = s.S != s.S, none = s.m == kNegInf && !bad;
  const float logS = none ? 0.0f : logf(s.S);
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (a.entropy) a.entropy[r] = bad ? nan : none ? 0.0f : logS - s.U / s.S;
    if (a.lp) a.lp[r] = !ok ? 0.0f : bad ? nan : none ? kNegInf : (xt - s.m) - logS;
    if (a.rank) a.rank[r] = ok ? s.ahead : -1;
  }
  if (lane < a.n_top) {
    const long at = (long)r * a.n_top + lane;
    const uint32_t o = (uint32_t)(key >> 32);
    if (a.top_id) a.top_id[at] = o ? (int32_t)~(uint32_t)key : -1;
    if (a.top_lp)
      a.top_lp[at] = !o ? kNegInf : bad ? nan : none ? kNegInf : (value_of(o) - s.m) - logS;
  }
}

// VEC: rows of 16-byte alignment, four logits a load.  TOP: with alternatives.
// RANK: with the target's rank.
template <bool VEC, bool TOP, bool RANK>
__global__ __launch_bounds__(256, 4) void k_logprobs(LogprobArgs a) {
  __shared__ u64 buf[TOP ? kLpWaves : 1][TOP ? kBuf : 1];
  __shared__ Sums ss[kLpWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = blockIdx.x / a.splits, z = blockIdx.x % a.splits;
  const float* x = a.x + r * a.stride;
  const int begin = z * a.chunk;
  const int end = z == a.splits - 1 || a.vocab - begin < a.chunk ? a.vocab : begin + a.chunk;
  // Place of a lane's j-th logit in a segment.  Logits are read once: no line of theirs is
  // worth keeping (512 x 151936 of them: 62 us, 66 with plain loads).
  auto place = [&](int j) { return VEC ? (j >> 2) * 256 + lane * 4 + (j & 3) : j * 64 + lane; };
  auto load = [&](float (&f)[16], int at) {
    if (at + kSeg <= end) {
#pragma unroll
      for (int j = 0; j < 16; j += VEC ? 4 : 1) {
        if (VEC) {
          const f32x4 v =
              __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(x + at + place(j)));
          f[j] = v.x;
          f[j + 1] = v.y;
          f[j + 2] = v.z;
          f[j + 3] = v.w;
        } else {
          f[j] = __builtin_nontemporal_load(x + at + place(j));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++) f[j] = at + place(j) < end ? x[at + place(j)] : kNegInf;
    }
  };
  float f[16];
  int at = begin + wave * kSeg;
  if (at < end) load(f, at);
  int target = -1;
  float xt = INFINITY, raw = 0.0f;
  if (a.targets) {
    target = a.targets[r];
    if ((unsigned)target < (unsigned)a.vocab) {
      raw = x[target];
      xt = fmaxf(raw, kNegInf);
    } else {
      target = -1;
    }
  }
  // the largest number below xt: ahead of the target is what is above it, at a lower place
  // also what equals it
  const int xb = __builtin_bit_cast(int, xt + 0.0f);
  const float below = __builtin_bit_cast(float, xb == 0 ? (int)0x80000001 : xb < 0 ? xb + 1 : xb - 1);
  Sums s = {kNegInf, 0.0f, 0.0f, 0};
  int ahead = 0;  // of the wave
  Best best = {0, 0, 0, kNegInf, false};
  for (; at < end; at += kLpWaves * kSeg) {
    float mx = kNegInf;
#pragma unroll
    for (int j = 0; j < 16; j++) mx = fmaxf(mx, f[j]);  // passes over NaN
    if (TOP) {
      const int hits = best.bound ? __popcll(__ballot(mx > best.value)) : 64;
      if (hits > 16) {
        uint32_t o[16];
#pragma unroll
        for (int j = 0; j < 16; j++)
          o[j] = at + place(j) < end ? order_of(fmaxf(f[j], kNegInf)) : 0u;
        best_add(best, o, a.n_top, buf[TOP ? wave : 0], [&](int j) { return at + place(j); });
      } else if (hits) {
        // few lanes: what is above the bound goes to the buffer, at most 256 more
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const u64 v = __ballot(f[j] > best.value);
          if (v) {
            if (f[j] > best.value)
              buf[TOP ? wave : 0][best.count + __popcll(v & ((1ull << lane) - 1))] =
                  (u64)order_of(f[j]) << 32 | (uint32_t)~(at + place(j));
            best.count += __popcll(v);
          }
        }
        if (best.count >= 64) {
          best_flush(best, a.n_top, buf[TOP ? wave : 0]);
          best.value = value_of(best.bound);
        }
      }
    }
    const float m = fmaxf(s.m, mx), ref = m == kNegInf ? 0.0f : m;
    // The segment's 16 terms first, then onto the lane's: one after the other, terms below half of
    // the last place of a large sum would all be lost.
    float S = 0.0f, U = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const float d = __builtin_elementwise_maximum(f[j] - ref, kFar);  // keeps NaN
      const float p = exp_of(d);
      S += p;
      U = __builtin_fmaf(p, d, U);
    }
    const float d = fmaxf(s.m - ref, kFar), e = exp_of(d);
    s.U = __builtin_fmaf(__builtin_fmaf(s.S, d, s.U), e, U);
    s.S = __builtin_fmaf(s.S, e, S);
    s.m = m;
    if (RANK) {  // last: the target's logit takes two loads, one after the other
      if (target >= at && target < at + kSeg) {
#pragma unroll
        for (int j = 0; j < 16; j++)
          ahead += __popcll(__ballot(
              f[j] > xt || (at + place(j) < target && (f[j] == xt || xt == kNegInf))));
      } else if (xt == kNegInf && target > at) {
        ahead += kSeg;  // a NaN counts as -inf
      } else {
        const float least = target > at ? below : xt;
#pragma unroll
        for (int j = 0; j < 16; j++) ahead += __popcll(__ballot(f[j] > least));
      }
    }
    if (at + kLpWaves * kSeg < end) load(f, at + kLpWaves * kSeg);
  }
  s = wave_join(s);
  s.ahead = ahead;
  if (lane == 0) ss[wave] = s;
  // The waves' lists into one of those at or above the largest bound.
  u64 key = 0;
  uint32_t bound = 0;
  if (TOP) {
    __shared__ uint32_t sb[kLpWaves];
    __shared__ int sc[kLpWaves];
    if (best.count > 0) {
      if (best.sorted) {
        best_flush(best, a.n_top, buf[wave]);
      } else {
        __builtin_amdgcn_wave_barrier();
        best.key = lane < best.count ? buf[wave][lane] : 0;
      }
    }
    if (lane == 0) sb[wave] = best.bound;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kLpWaves; w++) bound = sb[w] > bound ? sb[w] : bound;
    const bool in = (uint32_t)(best.key >> 32) >= (bound ? bound : 1u);
    const u64 v = __ballot(in);
    if (lane == 0) sc[wave] = __popcll(v);
    __syncthreads();
    int first = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kLpWaves; w++) {
      first += w < wave ? sc[w] : 0;
      all += sc[w];
    }
    if (in) buf[0][first + __popcll(v & ((1ull << lane) - 1))] = best.key;
    __syncthreads();
    if (wave == 0) {
      key = choose<kLpWaves>(buf[0], all, a.n_top);
      if (a.splits == 1) key = sort64(key);
    }
  } else {
    __syncthreads();
  }
  if (wave) return;
#pragma unroll 1
  for (int w = 1; w < kLpWaves; w++) s = join(s, ss[w]);
  if (a.splits == 1) {
    finish(a, r, s, key, target >= 0, raw);
    return;
  }
  const size_t part = (size_t)r * a.splits + z;
  if (TOP) a.keys[part * 64 + lane] = key;
  if (lane == 0) {
    *reinterpret_cast<float4*>(a.stats + 4 * part) =
        make_float4(s.m, s.S, s.U, __builtin_bit_cast(float, s.ahead));
  }
}

// The parts of a row joined.  The n-th largest of the lists' largest keys bounds what
// can be among the best n: no more than n lists have any such key, and with many lists not many
// more than n keys are left.  They are gathered in LDS and one wave chooses; where
// there are fewer lists than n, all their keys fit it.
//
// W: waves, one for up to kFew parts.
template <int W>
__global__ __launch_bounds__(64 * W) void k_logprobs_join(LogprobArgs a) {
  __shared__ u64 cand[W == 1 ? 64 * kFew : kChoose];
  __shared__ u64 head[W == 1 ? kFew : kMaxLists];
  __shared__ Sums ss[W];
  __shared__ int count;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x;
  const int lists = a.n_top > 0 ? a.splits : 0;
  const u64* keys = a.keys + (size_t)r * a.splits * 64;
  constexpr int kAhead = 4;  // all lists of a row of up to 262144 logits at once
  u64 k[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int i = i0 + j * W;
      k[j] = i < lists ? keys[(size_t)i * 64 + lane] : 0;
    }
  };
  load(wave);
  const int target = a.targets ? a.targets[r] : -1;
  const bool ok = (unsigned)target < (unsigned)a.vocab;
  const float xt = ok ? a.x[r * a.stride + target] : 0.0f;
  Sums s = {kNegInf, 0.0f, 0.0f, 0};
  for (int z = threadIdx.x; z < a.splits; z += 64 * W) {
    const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * ((size_t)r * a.splits + z));
    s = join(s, Sums{st.x, st.y, st.z, __builtin_bit_cast(int, st.w)});
  }
  if (threadIdx.x == 0) count = 0;
  if (wave * 64 < a.splits) {
    s = wave_join(s);
    if (lane == 0) ss[wave] = s;
  }
  u64 key = 0;
  if (lists) {
    u64 bound = 1;
    if (lists >= a.n_top) {
      for (int i0 = wave; i0 < lists; i0 += kAhead * W) {
        if (i0 > wave) load(i0);
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          const int i = i0 + j * W;
          if (i >= lists) break;
          const u64 h = largest64(k[j]);
          if (lane == 0) head[i] = h;
        }
      }
      __syncthreads();
      // each wave for itself
      u64 h = sort64(lane < lists ? head[lane] : 0);
      for (int i = 64; i < lists; i += 64)
        h = merge64(h, sort64(i + lane < lists ? head[i + lane] : 0));
      h = __shfl(h, a.n_top - 1);
      bound = h > bound ? h : bound;
      if (lists > kAhead * W) load(wave);
    }
    __syncthreads();
    for (int i0 = wave; i0 < lists; i0 += kAhead * W) {
      if (i0 > wave) load(i0);
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const bool in = k[j] >= bound;
        const u64 v = __ballot(in);
        if (!v) continue;
        int at = 0;
        if (lane == 0) at = atomicAdd(&count, __popcll(v));
        at = __builtin_amdgcn_readfirstlane(at) + __popcll(v & ((1ull << lane) - 1));
        if (in) cand[at] = k[j];
      }
    }
    __syncthreads();
    if (wave == 0)
      key = sort64(W == 1 || count <= 512 ? choose<8>(cand, count, a.n_top)
                                          : choose<0>(cand, count, a.n_top));
  } else {
    __syncthreads();
  }
  if (wave) return;
  for (int w = 1; w * 64 < a.splits && w < W; w++) s = join(s, ss[w]);
  finish(a, r, s, key, ok, xt);
}

}  // namespace
}  // namespace qr

using namespace qr;

extern "C" int qr_logprobs(qr_ctx* c, const float* x, long stride, int rows, int vocab,
                           const int32_t* targets, float* lp, float* entropy, int32_t* rank,
                           int n_top, int32_t* top_id, float* top_lp) {
  const char* who = "qr_logprobs";
  if (!c) return set_error(QR_ERR_INVALID, "%s: null ctx", who);
  if (rows < 0 || rows > 1 << 23 || vocab <= 0 || vocab > 1 << 30 || stride < vocab)
    return set_error(QR_ERR_INVALID, "%s: %d rows of %d logits, stride %ld", who, rows, vocab,
                     stride);
  if (n_top < 0 || n_top > QR_LOGPROBS_MAX_TOP)
    return set_error(QR_ERR_INVALID, "%s: n_top %d (0..%d)", who, n_top, QR_LOGPROBS_MAX_TOP);
  if (rows == 0) return QR_OK;
  if (!x) return set_error(QR_ERR_INVALID, "%s: null logits", who);
  if ((lp || rank) && !targets) return set_error(QR_ERR_INVALID, "%s: null targets", who);
  if ((uintptr_t)x & 3) return set_error(QR_ERR_INVALID, "%s: logits alignment", who);
  if (!top_id && !top_lp) n_top = 0;
  const hipError_t e0 = hipSetDevice(ctx_device(c));
  if (e0 != hipSuccess) return set_error(QR_ERR_HIP, "hipSetDevice: %s", hipGetErrorString(e0));
  LogprobArgs a = {x, stride, rows, vocab, targets, lp, entropy, rank, n_top, top_id, top_lp,
                   1, 0, nullptr, nullptr};
  // Parts: four workgroups per CU, each of at least a segment a wave.
  const int segs = (int)(((long)vocab + kLpWaves * kSeg - 1) / (kLpWaves * kSeg));
  long splits = (1024 + rows - 1) / rows;
  if (splits > segs) splits = segs;
  if (splits > kMaxLists) splits = kMaxLists;
  a.chunk = (int)((segs + splits - 1) / splits) * kLpWaves * kSeg;
  a.splits = (int)(((long)vocab + a.chunk - 1) / a.chunk);
  if (a.splits > 1) {
    const size_t parts = (size_t)rows * a.splits;
    void* w = nullptr;
    const size_t lists = n_top > 0 ? parts : 0;
    const int rc = ctx_scratch_get(c, parts * 16 + lists * 64 * sizeof(u64), who, &w);
    if (rc) return rc;
    a.stats = static_cast<float*>(w);
    a.keys = reinterpret_cast<u64*>(a.stats + 4 * parts);
  }
  const bool vec = !((uintptr_t)x & 15) && !(stride & 3);
  const dim3 grid((unsigned)((long)rows * a.splits));
  hipStream_t st = ctx_stream(c);
#define LP(V, T, R) hipLaunchKernelGGL((k_logprobs<V, T, R>), grid, dim3(256), 0, st, a)
  switch ((vec ? 4 : 0) | (n_top > 0 ? 2 : 0) | (rank ? 1 : 0)) {
    case 0: LP(false, false, false); break;
    case 1: LP(false, false, true); break;
    case 2: LP(false, true, false); break;
    case 3: LP(false, true, true); break;
    case 4: LP(true, false, false); break;
    case 5: LP(true, false, true); break;
    case 6: LP(true, true, false); break;
    default: LP(true, true, true); break;
  }
#undef LP
  if (a.splits > kFew)
    hipLaunchKernelGGL(k_logprobs_join<16>, dim3(rows), dim3(1024), 0, st, a);
  else if (a.splits > 1)
    hipLaunchKernelGGL(k_logprobs_join<1>, dim3(rows), dim3(64), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(QR_ERR_HIP, "k_logprobs: %s", hipGetErrorString(e));
  return QR_OK;
}
