// qr_kv_attn.hip -- attention of a ragged batch over a shared 8-bit KV pool
// (qr_kv_pool_attention), both products on int8 MFMA in fp32 accuracy.
//
// For a query row q and the cached k_t = ks_b kq_t, v_t = vs_b vq_t (int8
// values, one scale per block b of 16 tokens):
//   s_t = scale q . k_t,  out = sum_t exp(s_t) v_t / sum_t exp(s_t).
// The cache's operands are int8 already.  The other operand of each product is
// an fp32 number, which three int8 digits hold: x = u (65536 d2 + 256 d1 + d0),
// d in -128 .. 127, with u chosen by the row's (q) or the tile's (weights)
// largest value.  A product is then three exact integer products of 8 bits, and
// what it loses is the digits' last place, 2^-23 of the largest value: no less
// than fp32 products in fp32 sums keep.  The three products run on
// v_mfma_i32_16x16x64_i8 at twice the rate of bf16 and read the cache's bytes
// as they lie, so nothing is dequantized on the way.
//
// A wave serves 16 rows (queries times the query heads of a kv head) and takes
// 64 tokens a step.  Its four lane groups g = lane / 16 own a block each:
//   scores: A = 16 tokens of K in four tiles, tile t's row 4 g + i being token
//   16 g + 4 t + i; B = the rows' digits.  D then leaves row lane % 16 the four
//   tokens 4 t .. 4 t + 3 of block g, over the four tiles all 16 of them.
//   values: A = 16 columns of V, whose 16 bytes are a block's 16 tokens of a
//   column; B = the digits of the weights, in the lanes and bytes where the scores
//   left them.  No value crosses a lane between the two products, and the scales
//   of a block are one pair of numbers per lane.
//
// The weights carry V's scale: with vs = f 2^e (1 <= f < 2), w_t = f 2^(s_t
// log2(e) + e - M) against the running maximum M of the exponents, so the
// digits are taken from the numbers that are summed; the denominator adds the
// same powers times 2^-e.  Both are exact but for exp2.
#include <math.h>

#include "qr_kv_pool.h"

namespace qr {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;   // rows of a tile
constexpr int kStep = 64;   // tokens of a wave's step
constexpr int kWaves = 4;   // of a workgroup, taking the steps of its tokens in turn
constexpr float kNone = -INFINITY;
// Weights below 2 become whole numbers below 2^23 - 0x8080: added to 2^23 +
// 0x8080 they are the low mantissa bits of a float, and its three low bytes the
// digits but for the 0x80 that the two lower bytes carry.
constexpr float kWMul = 4177800.0f;
constexpr float kWAdd = 8388608.0f + 32896.0f;
constexpr float kQMax = 8355711.0f;  // 127 * (65536 + 256 + 1)
// Exponent of V scales that are 0 or smaller than it: such a block's weights
// lead no others, and its tokens still count in the denominator (at 2^60).
constexpr int kMinExp = -60;

// Where the rows of tile `slot` come from.
struct Tile {
  int row0;      // first query row
  int queries;   // of the tile, 0: none
  int seq, len;
  int pos0;      // position of the first
};

struct AttnArgs {
  PoolView p;
  Ragged r;
  const float* q;
  float* out;
  long q_stride, out_stride;
  int n_heads, group;   // query heads, query heads per kv head
  int hgroups, hpt;     // groups of at most 16 of a kv head's query heads, heads of each
  int qpt;              // queries of a tile
  int slots, splits;    // tiles of a head group, parts that a tile's tokens are cut into
  int chunk;            // tokens of a part, a multiple of kStep
  int window;
  float scale2;         // scale * log2(e)
  float* part;          // [tile, head][splits][kRows][hd], then [..][kRows][2]
  float* ml;
};

__device__ inline Tile tile_of(const AttnArgs& a, int slot) {
  Tile t;
  t.queries = 0;
  int piece;
  const int i = slot_seq(a.r, slot, a.qpt, 1, &piece);
  const SeqRows s = seq_rows(a.p, a.r, i);
  const int at = piece * a.qpt;
  if (piece < 0 || at >= s.m) return t;
  t.row0 = s.row0 + at;
  t.queries = s.m - at < a.qpt ? s.m - at : a.qpt;
  t.seq = s.seq;
  t.len = s.len;
  t.pos0 = s.len - s.m + at;
  return t;
}

// Tokens [*lo, *hi) that any row of the tile sees, *lo down to a step.
__device__ inline void tile_range(const AttnArgs& a, const Tile& t, int* lo, int* hi) {
  *hi = t.pos0 + t.queries;  // <= len
  if (*hi < 0) *hi = 0;
  int l = a.window > 0 ? t.pos0 - a.window + 1 : 0;
  if (l < 0) l = 0;
  *lo = l & ~(kStep - 1);
}

// Tokens of part z: a.chunk of them, all that is left in the last.
__device__ inline void part_range(const AttnArgs& a, int lo, int hi, int z, int* b, int* e) {
  const long s = (long)lo + (long)z * a.chunk;
  *b = s < hi ? (int)s : hi;
  *e = z == a.splits - 1 || s + a.chunk > hi ? hi : (int)(s + a.chunk);
  if (*e < *b) *e = *b;
}

__device__ inline uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}

// Four numbers whose bytes 0 and 1 carry 0x80 -> their digits, four to a dword.
__device__ inline void digits4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int* d0, int* d1,
                               int* d2) {
  const uint32_t lo = perm(b, a, 0x05010400u), hi = perm(d, c, 0x05010400u);
  *d0 = (int)(perm(hi, lo, 0x05040100u) ^ 0x80808080u);
  *d1 = (int)(perm(hi, lo, 0x07060302u) ^ 0x80808080u);
  const uint32_t l2 = perm(b, a, 0x0c0c0602u), h2 = perm(d, c, 0x0c0c0602u);
  *d2 = (int)perm(h2, l2, 0x05040100u);
}

__device__ inline v4i mfma(v4i a, v4i b, v4i c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// 65536 d2 + 256 d1 + d0 of three products, rounded to fp32 (the first two sum
// up below 2^31 over 64 tokens or 256 columns).
__device__ inline float joined(int s2, int s1, int s0) {
  return __builtin_fmaf((float)(s2 * 256 + s1), 256.0f, (float)s0);
}

// Over the four lane groups of a row.
__device__ inline float rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float rows_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ inline int4 load16(const int8_t* p) { return *reinterpret_cast<const int4*>(p); }
__device__ inline v4i as_v4(int4 x) { return v4i{x.x, x.y, x.z, x.w}; }

// out = sum over the parts of w_s O_s / L, in O_s' own maximum: the joining of
// two sums (m, l, o) and (m2, l2, o2).
__device__ inline float lift(float m, float to) {
  return m == kNone ? 0.0f : __builtin_amdgcn_exp2f(m - to);
}

template <int HD>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void k_pool_attn(AttnArgs a) {
  constexpr int NC = (HD + 63) / 64;  // 64-column chunks of a K row
  constexpr int NV = HD / 16;         // 16-column tiles of V
  __shared__ float so[2][kRows][HD + 4];
  __shared__ float sm[2][kRows][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.splits, z = blockIdx.x % a.splits, hy = blockIdx.y;
  const int kvh = hy / a.hgroups, hg = hy % a.hgroups;
  const Tile t = tile_of(a, slot);
  if (t.queries == 0) return;
  int lo, hi, tb, te;
  tile_range(a, t, &lo, &hi);
  part_range(a, lo, hi, z, &tb, &te);
  if (tb >= te && a.splits > 1) return;  // the joining launch skips it too

  // this lane's row
  const int qi = n / a.hpt, hh = hg * a.hpt + n % a.hpt;
  const bool row_ok = qi < t.queries && qi < a.qpt && hh < a.group;
  const long row = t.row0 + qi;
  const int head = kvh * a.group + hh;
  int row_hi = row_ok ? t.pos0 + qi + 1 : 0;
  int row_lo = row_ok && a.window > 0 ? row_hi - a.window : 0;
  // positions before 0 see nothing
  if (row_hi < 0) row_hi = 0;

  // q's digits: the lane holds columns 64 c + 16 g .. + 15 of its row
  v4i q0[NC], q1[NC], q2[NC];
  float qs;
  {
    float x[NC][16], amax = 0.0f;
    bool fine = true;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float4 f = make_float4(0, 0, 0, 0);
        if (row_ok && (HD % 64 == 0 || 64 * c + 16 * g < HD))
          f = *reinterpret_cast<const float4*>(a.q + row * a.q_stride + (long)head * HD + 64 * c +
                                               16 * g + 4 * j);
        x[c][4 * j] = f.x;
        x[c][4 * j + 1] = f.y;
        x[c][4 * j + 2] = f.z;
        x[c][4 * j + 3] = f.w;
      }
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int j = 0; j < 16; j++) {
        const float f = fabsf(x[c][j]);
        fine = fine && f <= 3.402823466e+38f;
        amax = fmaxf(amax, f);
      }
    amax = rows_max(amax);
    const float bad = rows_max(fine ? 0.0f : 1.0f);
    // below 2^-96 a row's scores are 0 beside any scale of K that fp32 values give
    amax = fmaxf(amax, 1.2621774e-29f);
    const float inv = kQMax / amax;
    qs = bad > 0.0f ? NAN : amax / kQMax * a.scale2;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float f = fminf(fmaxf(x[c][4 * j + i] * inv, -kQMax), kQMax);
          u[i] = (uint32_t)((int)rintf(f) + 0x8080);
        }
        int e0, e1, e2;
        digits4(u[0], u[1], u[2], u[3], &e0, &e1, &e2);
        q0[c][j] = e0;
        q1[c][j] = e1;
        q2[c][j] = e2;
      }
  }

  float o[NV][4];
#pragma unroll
  for (int d = 0; d < NV; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) o[d][i] = 0.0f;
  float M = kNone, L = 0.0f;

  const int kb = n >> 2;  // the block of the lane's K rows
  const int8_t* const data = a.p.data;
  // The lane's blocks of a step: kp / vp pages of K's and V's, -1 where there is none.
  auto pages = [&](int T0, int* kp, int* vp) {
    *kp = T0 + 16 * kb < te ? page_at(a.p, t.seq, (T0 + 16 * kb) >> a.p.page_shift) : -1;
    *vp = T0 + 16 * g < te ? page_at(a.p, t.seq, (T0 + 16 * g) >> a.p.page_shift) : -1;
  };
  const int pmask = (1 << (a.p.page_shift - 4)) - 1;
  int4 kr[4][NC];
  float2 sc;
  auto load_k = [&](int T0, int kp, int vp) {
    const size_t bk = kp < 0 ? 0 : block_at(a.p, kp, kvh, ((T0 >> 4) + kb) & pmask);
    const size_t bv = vp < 0 ? 0 : block_at(a.p, vp, kvh, ((T0 >> 4) + g) & pmask);
    const int8_t* s = data + bk * (2 * kKvBlock * HD) + (n & 3) * HD + 16 * g;
#pragma unroll
    for (int tt = 0; tt < 4; tt++)
#pragma unroll
      for (int c = 0; c < NC; c++)
        if (HD % 64 == 0 || 64 * c + 16 * g < HD)
          kr[tt][c] = load16(s + 4 * tt * HD + 64 * c);
        else
          kr[tt][c] = make_int4(0, 0, 0, 0);
    sc = make_float2(0.0f, 0.0f);
    if (vp >= 0) sc = *reinterpret_cast<const float2*>(a.p.scale + 2 * bv);
  };

  int T0 = tb + wave * kStep;
  int kp, vp, kp1 = -1, vp1 = -1;
  if (T0 < te) {
    pages(T0, &kp, &vp);
    load_k(T0, kp, vp);
    pages(T0 + kWaves * kStep, &kp1, &vp1);
  }
  for (; T0 < te; T0 += kWaves * kStep) {
    // V of this step
    int4 vr[NV];
    {
      const size_t bv = vp < 0 ? 0 : block_at(a.p, vp, kvh, ((T0 >> 4) + g) & pmask);
      const int8_t* s = data + bv * (2 * kKvBlock * HD) + kKvBlock * HD + n * kKvBlock;
#pragma unroll
      for (int d = 0; d < NV; d++) vr[d] = load16(s + d * 16 * kKvBlock);
    }
    // scores
    v4i s0[4], s1[4], s2[4];
#pragma unroll
    for (int tt = 0; tt < 4; tt++) {
      s0[tt] = s1[tt] = s2[tt] = v4i{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const v4i k = as_v4(kr[tt][c]);
        s0[tt] = mfma(k, q0[c], s0[tt]);
        s1[tt] = mfma(k, q1[c], s1[tt]);
        s2[tt] = mfma(k, q2[c], s2[tt]);
      }
    }
    const float ks = sc.x, vs = sc.y;
    const bool here = vp >= 0;
    const int vblk = T0 + 16 * g;
    // the next step's K behind this one's V, its pages known a step ahead
    const int Tn = T0 + kWaves * kStep;
    vp = vp1;
    if (Tn < te) {
      load_k(Tn, kp1, vp1);
      pages(Tn + kWaves * kStep, &kp1, &vp1);
    }
    // exponents: scores in powers of two, with V's
    int ev = kMinExp;
    if (vs > 0x1p-60f) ev = (int)((__builtin_bit_cast(uint32_t, vs) >> 23) & 255) - 127;
    const float f = here ? vs * __builtin_bit_cast(float, (uint32_t)(127 - ev) << 23) : 0.0f;
    const float back = __builtin_bit_cast(float, (uint32_t)(127 - ev) << 23);
    const float c = qs * ks, evf = (float)ev;
    float e[16], mx = kNone;
#pragma unroll
    for (int tt = 0; tt < 4; tt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int tok = vblk + 4 * tt + i;
        float v = __builtin_fmaf(joined(s2[tt][i], s1[tt][i], s0[tt][i]), c, evf);
        if (!(here && tok < row_hi && tok >= row_lo && tok < te)) v = kNone;
        e[4 * tt + i] = v;
        mx = fmaxf(mx, v);
      }
    mx = rows_max(mx);
    const float to = fmaxf(M, mx);
    const float ref = to == kNone ? 0.0f : to;
    const float alpha = lift(M, ref);
    M = to;
    float sum = 0.0f;
    v4i p0, p1, p2;
    const float fw = f * kWMul;
#pragma unroll
    for (int tt = 0; tt < 4; tt++) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float p = __builtin_amdgcn_exp2f(e[4 * tt + i] - ref);
        sum += p;
        u[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(p, fw, kWAdd));
      }
      int e0, e1, e2;
      digits4(u[0], u[1], u[2], u[3], &e0, &e1, &e2);
      p0[tt] = e0;
      p1[tt] = e1;
      p2[tt] = e2;
    }
    L = __builtin_fmaf(sum, back, L * alpha);
    // values
#pragma unroll
    for (int d = 0; d < NV; d++) {
      const v4i zero = v4i{0, 0, 0, 0}, v = as_v4(vr[d]);
      const v4i a0 = mfma(v, p0, zero), a1 = mfma(v, p1, zero), a2 = mfma(v, p2, zero);
#pragma unroll
      for (int i = 0; i < 4; i++)
        o[d][i] = __builtin_fmaf(o[d][i], alpha, joined(a2[i], a1[i], a0[i]));
    }
  }
  L = rows_sum(L);

  // join the waves: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
  for (int half = 2; half; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int d = 0; d < NV; d++)
        *reinterpret_cast<float4*>(&so[wave - half][n][16 * d + 4 * g]) =
            make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
      if (g == 0) {
        sm[wave - half][n][0] = M;
        sm[wave - half][n][1] = L;
      }
    }
    __syncthreads();
    if (wave < half) {
      const float M2 = sm[wave][n][0], L2 = sm[wave][n][1];
      const float to = fmaxf(M, M2), ref = to == kNone ? 0.0f : to;
      const float x = lift(M, ref), y = lift(M2, ref);
      L = L * x + L2 * y;
#pragma unroll
      for (int d = 0; d < NV; d++) {
        const float4 w = *reinterpret_cast<const float4*>(&so[wave][n][16 * d + 4 * g]);
        o[d][0] = o[d][0] * x + w.x * y;
        o[d][1] = o[d][1] * x + w.y * y;
        o[d][2] = o[d][2] * x + w.z * y;
        o[d][3] = o[d][3] * x + w.w * y;
      }
      M = to;
    }
    __syncthreads();
  }
  if (wave != 0 || !row_ok) return;
  if (a.splits == 1) {
    // a row that saw nothing: L = 0
    const float inv = L == 0.0f ? 0.0f : 1.0f / (L * kWMul);
    float* dst = a.out + row * a.out_stride + (long)head * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < NV; d++)
      *reinterpret_cast<float4*>(dst + 16 * d) =
          make_float4(o[d][0] * inv, o[d][1] * inv, o[d][2] * inv, o[d][3] * inv);
  } else {
    const size_t at = ((size_t)(slot * gridDim.y + hy) * a.splits + z) * kRows + n;
#pragma unroll
    for (int d = 0; d < NV; d++)
      *reinterpret_cast<float4*>(a.part + at * HD + 16 * d + 4 * g) =
          make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    if (g == 0) {
      a.ml[2 * at] = M;
      a.ml[2 * at + 1] = L;
    }
  }
}

// The parts of each row joined: a workgroup per row, a thread per column (and
// a group of threads per part where columns leave some).
template <int HD>
__global__ __launch_bounds__(256) void k_pool_attn_join(AttnArgs a) {
  __shared__ float red[256];
  const int n = blockIdx.x % kRows, slot = blockIdx.x / kRows, hy = blockIdx.y;
  const Tile t = tile_of(a, slot);
  const int qi = n / a.hpt, hh = hy % a.hgroups * a.hpt + n % a.hpt;
  if (!(qi < t.queries && hh < a.group)) return;
  int lo, hi;
  tile_range(a, t, &lo, &hi);
  int parts = 0;
  if (hi > lo) {
    parts = (int)(((long)hi - lo + a.chunk - 1) / a.chunk);
    if (parts > a.splits) parts = a.splits;
  }
  const size_t at = (size_t)(slot * gridDim.y + hy) * a.splits * kRows + n;
  float M = kNone;
  for (int s = threadIdx.x; s < parts; s += 256) M = fmaxf(M, a.ml[2 * (at + (size_t)s * kRows)]);
  for (int d = 32; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = M == kNone ? 0.0f : M;
  __syncthreads();
  constexpr int kGroups = 256 / HD > 0 ? 256 / HD : 1;
  const int c = threadIdx.x % HD, grp = threadIdx.x / HD;
  float sum = 0.0f, L = 0.0f;
  if (grp < kGroups)
    for (int s = grp; s < parts; s += kGroups) {
      const size_t r = at + (size_t)s * kRows;
      const float w = lift(a.ml[2 * r], ref);
      sum += w * a.part[r * HD + c];
      L += w * a.ml[2 * r + 1];
    }
  if (kGroups > 1) {
    __shared__ float redl[256];
    red[threadIdx.x] = sum;
    redl[threadIdx.x] = L;
    __syncthreads();
    if (grp == 0)
      for (int j = 1; j < kGroups; j++) {
        sum += red[j * HD + c];
        L += redl[j * HD + c];
      }
  }
  if (grp == 0)
    a.out[(t.row0 + qi) * a.out_stride + (long)(hy / a.hgroups * a.group + hh) * HD + c] =
        L == 0.0f ? 0.0f : sum / (L * kWMul);
}

// How the work is cut.  Heads: at most 16 of a kv head's query heads share a
// tile, as many queries beside each other as fill it.  Tokens: a tile's part is
// one workgroup; there are as many parts as it takes to have four workgroups
// per CU (two are resident; lengths differ), each of 256 tokens or more.
AttnArgs attn_plan(const PoolView& p, const Ragged& r, int n_heads, int max_len, int window) {
  AttnArgs a = {};
  a.p = p;
  a.r = r;
  a.n_heads = n_heads;
  a.group = n_heads / p.n_kv_heads;
  a.hgroups = (a.group + kRows - 1) / kRows;
  a.hpt = (a.group + a.hgroups - 1) / a.hgroups;
  a.qpt = kRows / a.hpt;
  a.window = window;
  a.slots = r.T / a.qpt + r.n;
  long range = max_len;
  if (window > 0 && window + (long)a.qpt + kStep < range) range = window + (long)a.qpt + kStep;
  const long tiles = (r.T / a.qpt > r.n ? r.T / a.qpt : r.n) * (long)p.n_kv_heads * a.hgroups;
  long splits = (1024 + tiles - 1) / tiles;
  const long most = (range + 4 * kStep - 1) / (4 * kStep);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  long chunk = (range + splits - 1) / splits;
  chunk = (chunk + kStep - 1) / kStep * kStep;
  a.chunk = (int)chunk;
  a.splits = (int)((range + chunk - 1) / chunk);
  return a;
}

size_t part_floats(const AttnArgs& a) {
  return (size_t)a.slots * a.p.n_kv_heads * a.hgroups * a.splits * kRows;
}

}  // namespace

size_t kv_attention_scratch(const PoolView& p, const Ragged& r, int n_heads, int max_len,
                            int window) {
  const AttnArgs a = attn_plan(p, r, n_heads, max_len, window);
  return a.splits == 1 ? 0 : part_floats(a) * (p.hd + 2) * sizeof(float);
}

hipError_t kv_attention_launch(const PoolView& p, const Ragged& r, int n_heads, const float* q,
                               long q_stride, float* out, long out_stride, int max_len, int window,
                               float scale, void* work, hipStream_t st) {
  AttnArgs a = attn_plan(p, r, n_heads, max_len, window);
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.scale2 = scale * 1.44269504088896340736f;
  a.part = static_cast<float*>(work);
  a.ml = a.part + part_floats(a) * p.hd;
  const dim3 grid((unsigned)(a.slots * a.splits), (unsigned)(p.n_kv_heads * a.hgroups));
#define ATTN(HD)                                                                               \
  {                                                                                            \
    hipLaunchKernelGGL(k_pool_attn<HD>, grid, dim3(256), 0, st, a);                            \
    if (a.splits > 1)                                                                          \
      hipLaunchKernelGGL(k_pool_attn_join<HD>, dim3(kRows * a.slots, grid.y), dim3(256), 0, st, a); \
  }
  switch (p.hd) {
    case 32: ATTN(32) break;
    case 64: ATTN(64) break;
    case 96: ATTN(96) break;
    case 128: ATTN(128) break;
    case 160: ATTN(160) break;
    case 192: ATTN(192) break;
    case 224: ATTN(224) break;
    default: ATTN(256) break;
  }
#undef ATTN
  return hipGetLastError();
}

}  // namespace qr
