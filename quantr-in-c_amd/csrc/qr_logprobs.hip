// qr_logprobs.hip -- log probabilities of given tokens, entropy and the best
// alternatives of rows of logits (qr_logprobs of qr_hip.h), in one pass.
//
// With m = max x, S = sum e^(x - m) and U = sum e^(x - m) (x - m):
//   log p_t = (x_t - m) - log S,   -sum p log p = log S - U / S.
// A lane keeps its own m, S and U and lifts them when its maximum grows (S e^d,
// (U + S d) e^d with d the maximum's step down), so the row is read once, nothing
// is exchanged on the way, and the sums are 32-bit sums of few terms each.  The
// best tokens come from the same read: a wave keeps its 64 best as 64-bit
// keys (the logit's order, then the lower index), sorted over its lanes, and
// looks at a segment of 1024 logits only where one of them beats the n-th.
// Long rows are bound by HBM; few rows are cut into parts that a second launch
// joins, bound by latency.
#include <math.h>

#include "qr_internal.h"

namespace qr {
namespace {

constexpr int kSeg = 1024;   // logits of a wave's step: 16 a lane
constexpr int kLpWaves = 4;
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.44269504088896340736f;
// Below this a difference's exponential is 0 in fp32; it stands for -inf, whose
// product with 0 would be NaN.
constexpr float kFar = -200.0f;

typedef unsigned long long u64;

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
  float* stats;        // [row][part][4]: m, S, U, and the rank with the bad flag's bit
};

struct Sums {
  float m, S, U;
  int ahead;   // logits ahead of the target's
  int bad;     // a NaN or +inf among them
};

__device__ inline Sums join(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - r.m, kFar), db = fmaxf(b.m - r.m, kFar);
  const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
  r.S = a.S * fa + b.S * fb;
  r.U = (a.U + a.S * da) * fa + (b.U + b.S * db) * fb;
  r.ahead = a.ahead + b.ahead;
  r.bad = a.bad | b.bad;
  return r;
}

__device__ inline Sums wave_join(Sums s) {
  for (int d = 1; d < 64; d <<= 1) {
    Sums o;
    o.m = __shfl_xor(s.m, d);
    o.S = __shfl_xor(s.S, d);
    o.U = __shfl_xor(s.U, d);
    o.ahead = __shfl_xor(s.ahead, d);
    o.bad = __shfl_xor(s.bad, d);
    s = join(s, o);
  }
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

// One compare-exchange with the lane `d` away; keeps the larger where `up`.
__device__ inline u64 exchange(u64 k, int d, bool up) {
  const u64 o = __shfl_xor(k, d);
  return up == (o > k) ? o : k;
}
// 64 keys, descending over the lanes.
__device__ inline u64 sort64(u64 k) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int d = size / 2; d; d >>= 1) k = exchange(k, d, ((lane & d) == 0) == ((lane & size) == 0 || size == 64));
  return k;
}
// The 64 largest of two descending lists, descending.
__device__ inline u64 merge64(u64 a, u64 b) {
  const int lane = threadIdx.x & 63;
  const u64 r = __shfl(b, 63 - lane);
  u64 k = r > a ? r : a;
#pragma unroll
  for (int d = 32; d; d >>= 1) k = exchange(k, d, (lane & d) == 0);
  return k;
}

// A wave's best logits.
struct Best {
  u64 key;        // lane i: the i-th best, 0 where there are fewer
  uint32_t tau;   // order of the n-th best, 0 where there are fewer
  float tauf;     // its value, -inf where there are fewer
};

__device__ inline void best_done(Best& b, int n) {
  b.tau = (uint32_t)(__shfl(b.key, n - 1) >> 32);
  b.tauf = b.tau ? value_of(b.tau) : kNegInf;
}

// A segment's logits that beat the n-th best join the list.  o: their orders (0:
// no logit), idx0 + step(j): their places.  With more than 64 of them, those
// below the n-th largest of the lanes' maxima cannot be among the best n and
// are left out first (found bit by bit), so that at most 16 n are sorted but for
// equal ones.
template <class At>
__device__ inline void best_add(Best& b, const uint32_t (&o)[16], int n, u64* buf, At at) {
  const int lane = threadIdx.x & 63;
  int c = 0;
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    c += __popcll(__ballot(o[j] > b.tau));
    mx = o[j] > mx ? o[j] : mx;
  }
  uint32_t least = b.tau + 1;
  if (c > 64) {
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; bit--) {
      const uint32_t u = t | 1u << bit;
      if (__popcll(__ballot(mx >= u)) >= n) t = u;
    }
    if (t > least) least = t;
  }
  int count = 0;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    const u64 v = __ballot(o[j] >= least);
    if (o[j] >= least)
      buf[count + __popcll(v & ((1ull << lane) - 1))] = (u64)o[j] << 32 | (uint32_t)~at(j);
    count += __popcll(v);
  }
  __builtin_amdgcn_wave_barrier();
  for (int i = 0; i < count; i += 64) b.key = merge64(b.key, sort64(i + lane < count ? buf[i + lane] : 0));
  best_done(b, n);
}

// The row's results, by wave 0 with the whole row's sums and list.
__device__ inline void finish(const LogprobArgs& a, int r, const Sums& s, u64 key) {
  const int lane = threadIdx.x & 63;
  const bool none = s.m == kNegInf;
  const float logS = none ? 0.0f : logf(s.S);
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (a.entropy) a.entropy[r] = s.bad ? nan : none ? 0.0f : logS - s.U / s.S;
    if (a.lp || a.rank) {
      const int t = a.targets[r];
      const bool ok = (unsigned)t < (unsigned)a.vocab;
      if (a.lp) {
        float v = 0.0f;
        if (ok) v = s.bad ? nan : none ? kNegInf : (a.x[r * a.stride + t] - s.m) - logS;
        a.lp[r] = v;
      }
      if (a.rank) a.rank[r] = ok ? s.ahead : -1;
    }
  }
  if (lane < a.n_top) {
    const long at = (long)r * a.n_top + lane;
    const uint32_t o = (uint32_t)(key >> 32);
    if (a.top_id) a.top_id[at] = o ? (int32_t)~(uint32_t)key : -1;
    if (a.top_lp)
      a.top_lp[at] = !o ? kNegInf : s.bad ? nan : none ? kNegInf : (value_of(o) - s.m) - logS;
  }
}

// The waves' sums and lists into wave 0's.
__device__ inline void waves_join(Sums& s, u64& key, bool top) {
  __shared__ Sums ss[kLpWaves];
  __shared__ u64 sk[kLpWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) ss[wave] = s;
  if (top) sk[wave][lane] = key;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < kLpWaves; w++) {
    s = join(s, ss[w]);
    if (top) key = merge64(key, sk[w][lane]);
  }
}

// VEC: rows of 16-byte alignment, four logits a load.  TOP: with alternatives.
// RANK: with the target's rank.
template <bool VEC, bool TOP, bool RANK>
__global__ __launch_bounds__(256) void k_logprobs(LogprobArgs a) {
  __shared__ u64 buf[TOP ? kLpWaves : 1][TOP ? kSeg : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = blockIdx.x / a.splits, z = blockIdx.x % a.splits;
  const float* x = a.x + r * a.stride;
  const int begin = z * a.chunk;
  const int end = z == a.splits - 1 || a.vocab - begin < a.chunk ? a.vocab : begin + a.chunk;
  int target = -1;
  float xt = INFINITY;
  if (RANK) {
    target = a.targets[r];
    if ((unsigned)target < (unsigned)a.vocab) xt = fmaxf(x[target], kNegInf);
  }
  Sums s = {kNegInf, 0.0f, 0.0f, 0, 0};
  Best best = {0, 0, kNegInf};
  // place of a lane's j-th logit in a segment
  auto place = [&](int j) { return VEC ? (j >> 2) * 256 + lane * 4 + (j & 3) : j * 64 + lane; };
  float f[16];
  auto load = [&](int at) {
    if (at + kSeg <= end) {
#pragma unroll
      for (int j = 0; j < 16; j += VEC ? 4 : 1) {
        if (VEC) {
          const float4 v = *reinterpret_cast<const float4*>(x + at + place(j));
          f[j] = v.x;
          f[j + 1] = v.y;
          f[j + 2] = v.z;
          f[j + 3] = v.w;
        } else {
          f[j] = x[at + place(j)];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++) f[j] = at + place(j) < end ? x[at + place(j)] : kNegInf;
    }
  };
  int at = begin + wave * kSeg;
  if (at < end) load(at);
  for (; at < end; at += kLpWaves * kSeg) {
    float v[16];
    float mx = kNegInf;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      s.bad |= !(f[j] <= 3.402823466e+38f);
      v[j] = fmaxf(f[j], kNegInf);  // a NaN in its order
      mx = fmaxf(mx, v[j]);
    }
    if (at + kLpWaves * kSeg < end) load(at + kLpWaves * kSeg);
    {
      const float m = fmaxf(s.m, mx), d = fmaxf(s.m - m, kFar);
      const float e = __builtin_amdgcn_exp2f(d * kLog2e);
      s.U = (s.U + s.S * d) * e;
      s.S = s.S * e;
      s.m = m;
#pragma unroll
      for (int j = 0; j < 16; j++) {
        const float dj = fmaxf(v[j] - m, kFar);
        const float p = __builtin_amdgcn_exp2f(dj * kLog2e);
        s.S += p;
        s.U = __builtin_fmaf(p, dj, s.U);
      }
    }
    if (RANK) {
#pragma unroll
      for (int j = 0; j < 16; j++)
        s.ahead += v[j] > xt || (v[j] == xt && at + place(j) < target);
    }
    if (TOP && (best.tau == 0 || __ballot(mx > best.tauf))) {
      uint32_t o[16];
#pragma unroll
      for (int j = 0; j < 16; j++) o[j] = at + place(j) < end ? order_of(v[j]) : 0u;
      best_add(best, o, a.n_top, buf[TOP ? wave : 0], [&](int j) { return at + place(j); });
    }
  }
  s = wave_join(s);
  waves_join(s, best.key, TOP);
  if (wave) return;
  if (a.splits == 1) {
    finish(a, r, s, best.key);
    return;
  }
  const size_t p = (size_t)r * a.splits + z;
  if (TOP) a.keys[p * 64 + lane] = best.key;
  if (lane == 0) {
    float* st = a.stats + 4 * p;
    st[0] = s.m;
    st[1] = s.S;
    st[2] = s.U;
    st[3] = __builtin_bit_cast(float, s.ahead | s.bad << 31);
  }
}

__global__ __launch_bounds__(256) void k_logprobs_join(LogprobArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x;
  Sums s = {kNegInf, 0.0f, 0.0f, 0, 0};
  for (int z = threadIdx.x; z < a.splits; z += 256) {
    const float* st = a.stats + 4 * ((size_t)r * a.splits + z);
    const int w = __builtin_bit_cast(int, st[3]);
    s = join(s, Sums{st[0], st[1], st[2], w & 0x7FFFFFFF, (int)((uint32_t)w >> 31)});
  }
  u64 key = 0;
  if (a.n_top > 0)
    for (int z = wave; z < a.splits; z += kLpWaves)
      key = merge64(key, a.keys[((size_t)r * a.splits + z) * 64 + lane]);
  s = wave_join(s);
  waves_join(s, key, a.n_top > 0);
  if (wave == 0) finish(a, r, s, key);
}

}  // namespace
}  // namespace qr

using namespace qr;

extern "C" int qr_logprobs(qr_ctx* c, const float* x, long stride, int rows, int vocab,
                           const int32_t* targets, float* lp, float* entropy, int32_t* rank,
                           int n_top, int32_t* top_id, float* top_lp) {
  const char* who = "qr_logprobs";
  if (!c) return set_error(QR_ERR_INVALID, "%s: null ctx", who);
  if (rows < 0 || vocab <= 0 || stride < vocab)
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
  a.chunk = (int)((segs + splits - 1) / splits) * kLpWaves * kSeg;
  a.splits = (int)(((long)vocab + a.chunk - 1) / a.chunk);
  if (a.splits > 1) {
    const size_t parts = (size_t)rows * a.splits;
    void* w = nullptr;
    const int rc = ctx_scratch_get(c, parts * (64 * sizeof(u64) + 16), who, &w);
    if (rc) return rc;
    a.keys = static_cast<u64*>(w);
    a.stats = reinterpret_cast<float*>(a.keys + parts * 64);
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
  if (a.splits > 1) hipLaunchKernelGGL(k_logprobs_join, dim3(rows), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(QR_ERR_HIP, "k_logprobs: %s", hipGetErrorString(e));
  return QR_OK;
}
