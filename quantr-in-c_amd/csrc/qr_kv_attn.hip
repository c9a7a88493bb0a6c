// qr_kv_attn.hip -- attention of a ragged batch over a shared 8-bit KV pool
// (qr_kv_pool_attention), both products on MFMA.
//
// For a query row q and the cached k_t = ks_b kq_t, v_t = vs_b vq_t (int8
// values, one scale per block b of 16 tokens):
//   s_t = scale q . k_t,  out = sum_t exp(s_t) v_t / sum_t exp(s_t).
// The other operand of each product is an fp32 number, a row's q or a token's weight: two fp16
// pieces, the nearest one and 2048 times what it leaves, hold it to 2^-22 of itself (a score's
// own roundings in fp32 move a weight more) or 2^-50 of the largest of its row.  The cache's
// bytes are widened to fp16 on the way, 1.25 instructions each; products are exact and sums
// fp32, each piece's apart.  (Digits of the largest on int8 products, 40 us for a prompt's 512
// rows where this takes 47, gave the small ones up: beside a token that takes 0.9999 of the
// weight with values of 0 the output was off by a fifth of itself, beside a channel of q of 10^6
// by a fortieth.  Three bf16 pieces of the weights, which know no largest, took 50 us where
// two of fp16 took 44.)
//
// A workgroup of four waves serves a tile of 16 or 32 rows (queries times the query
// heads of a kv head) and takes 256 tokens a round, a wave 64 of them.  A wave's four
// lane groups g = lane / 16 own a block each:
//   scores: A = 16 tokens of K in four tiles, tile t's row 4 g + i being token
//   16 g + 4 t + i, eight of a lane's 16 columns to an instruction; B = the rows' pieces.  D
//   then leaves row lane % 16 the four tokens 4 t .. 4 t + 3 of block g, over the four tiles
//   all 16 of them.
//   values: A = 16 columns of V, whose 16 bytes are a block's 16 tokens of a
//   column, eight to an instruction; B = the weights' pieces, in the lanes where the scores
//   left them, so no weight crosses a lane.
// The values' columns are what the waves share out: each reads all four waves'
// pieces from LDS (16 KiB).  A wave that kept all columns of its own tokens instead converted four
// times as many sums, held 206 registers for 164, and ended in a join of the waves.
//
// What bounds it.  Many rows: neither unit alone (a prompt's 512 rows of 8 heads a kv head at
// 1501 .. 2012, 47 us: VALU issue 52 % of the time, matrix units 23 %); of a wave's time 30 % goes
// by waiting to issue beside the SIMD's other wave and 27 % at barriers and for memory.  A wave
// in its products goes before the other one, so that one's products run under the other's softmax
// (52 us without it).  One row a sequence: two launches' latency, the widening, and then HBM (32 of
// 587 .. 4096 tokens, 66 MB: 23.5 us; one of 702: 9.1).
//
// The weights carry V's scale: with vs = f 2^e (1/2 <= f < 1), w_t = f 2^(s_t
// log2(e) + e - M) against a reference M that brings the round's largest weight just
// below 1 (more than 2^kFall below the row's largest it does not follow), so the pieces are
// those of the numbers that are summed.  The denominator runs against the maximum N of the scores
// alone, its terms the same powers times 2^(M - e - N): values of V however unlike move no
// token out of it.
#include <math.h>

#include "qr_kv_pool.h"
#include "qr_lanes.h"

namespace qr {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;   // tokens of a wave's step
constexpr int kWaves = 4;   // of a workgroup
constexpr int kRound = kStep * kWaves;
constexpr int kPages = 1024;  // blocks whose pages are held at a time: 64 rounds
constexpr int kMaxParts = 1024;  // of a tile's tokens
constexpr long kMostItems = 32768;  // workgroups with parts: what they leave stays below 600 MB
constexpr int kJoinWave = 16;    // up to as many one wave joins a row
constexpr float kNone = -INFINITY;
// A number up to kTop as two fp16: the nearest one, and kSecond times what it leaves.
constexpr float kTop = 32768.0f, kSecond = 2048.0f;
// Exponent of V scales that are 0 or subnormal: such a block's weights lead no others.
constexpr int kMinExp = -125;
// A block whose exponents lie further below M takes its powers 2^-kDeep below them, so that
// they are there for the denominator.
constexpr float kDeep = 60.0f;
constexpr float kFall = 24.0f;

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
  int group;            // query heads per kv head
  int hgroups, hpt;     // groups of at most 16 of a kv head's query heads, heads of each
  int rt, qpt, extra;   // 16-row sets of a tile, queries of it, slots beyond T / qpt for each sequence
  int slots, splits;    // tiles of a head group, parts that a tile's tokens are cut into
  int chunk;            // tokens of a part, a multiple of kStep
  int window;
  float scale2;         // scale * log2(e)
  float* part;          // [tile, head][splits][row][hd], then [..][row][4]
  float* ml;
  int4* meta;           // [tile]: first row, queries, parts
};

// All but its length and positions, which tile_len adds.
__device__ inline Tile tile_of(const AttnArgs& a, int slot, SeqRows* s) {
  Tile t;
  int piece;
  *s = slot_rows(a.p, a.r, slot, a.qpt, a.extra, &piece);
  const int at = piece * a.qpt;
  t.row0 = s->row0 + at;
  t.queries = s->m - at < a.qpt ? s->m - at : a.qpt;
  if (piece < 0 || at >= s->m) t.queries = 0;
  t.seq = s->seq;
  return t;
}
__device__ inline void tile_len(const AttnArgs& a, const SeqRows& s, Tile* t) {
  t->len = seq_len(a.p, s);
  t->pos0 = t->len - s.m + (t->row0 - s.row0);
}

// Which tile and part a workgroup takes.  The last tiles, whose rows see most, come
// first.  Workgroups go round the 8 XCDs in order, and a sequence's later parts are
// empty where it is short, so neither the part nor the sequence may go with the
// XCD: part after part, the tiles of each turned by some (32 sequences of up to 4096
// tokens: 24.6 us, 35 with the eight parts of a tile side by side, every first part on one XCD).
__device__ inline void work_of(const AttnArgs& a, int* slot, int* z) {
  *z = (int)(blockIdx.x / a.slots);
  int s = (int)(blockIdx.x % a.slots);
  if (a.splits > 1) s = (s + *z + (*z >> 2) + (int)blockIdx.y) % a.slots;
  *slot = a.slots - 1 - s;
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

// Two numbers' pieces: a = p0 + p1 / kSecond to 2^-22 of a, or 2^-36 where that is more.
__device__ inline void pieces2(float a, float b, int* p0, int* p1) {
  const v2h h = __builtin_convertvector((v2f{a, b}), v2h);
  const v2f left = {__builtin_fmaf(-kSecond, (float)h.x, a * kSecond),
                    __builtin_fmaf(-kSecond, (float)h.y, b * kSecond)};
  *p0 = __builtin_bit_cast(int, h);
  *p1 = __builtin_bit_cast(int, __builtin_convertvector(left, v2h));
}

// Eight int8 as fp16, exactly: beside the byte 0x64 the unsigned x + 128 is the fp16 1024 + 128 + x.
__device__ inline v8h widened(int lo, int hi) {
  const uint32_t a = (uint32_t)lo ^ 0x80808080u, b = (uint32_t)hi ^ 0x80808080u;
  const v4i w = {(int)perm(0x64646464u, a, 0x05010400u), (int)perm(0x64646464u, a, 0x07030602u),
                 (int)perm(0x64646464u, b, 0x05010400u), (int)perm(0x64646464u, b, 0x07030602u)};
  return __builtin_bit_cast(v8h, w) - (_Float16)1152.0f;
}
__device__ inline v4f mfma(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ inline int4 load16(const int8_t* p) { return *reinterpret_cast<const int4*>(p); }

// The reference for weights up to 2^x: the next multiple of 1 / 16, so that the references'
// and V's exponents differ by what fp32 holds exactly and no rounding of theirs moves a
// whole block or row, above x by what rounding may have taken from x.  From kLarge on x itself.
constexpr float kLarge = 1048576.0f;
__device__ inline float reference(float x) {
  const float r = ceilf(__builtin_fmaf(fabsf(x), 0x1p-22f, x) * 16.0f) * 0.0625f;
  return fabsf(x) < kLarge ? r : x;
}

// The factor that takes a sum against maximum m to one against `to`.
__device__ inline float lift(float m, float to) {
  return m == kNone ? 0.0f : __builtin_amdgcn_exp2f(m - to);
}

// A sum against M over the denominator l against N; 0 for a row that saw nothing.  The whole
// powers of two come last, so that nothing on the way leaves the normal numbers.
struct Over {
  float inv;
  int exp;
  __device__ Over(float M, float N, float l) {
    const float d = M - N, whole = floorf(d);
    exp = (int)whole;
    inv = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(d - whole) / (l * kTop);
  }
  __device__ float operator()(float x) const { return __builtin_ldexpf(x * inv, exp); }
};

// Workgroups a CU: three of 16 rows up to head_dim 128, two otherwise; none spills (attn_plan
// counts on as many).
template <int HD, int RT>
__global__ __launch_bounds__(256, HD <= 128 && RT == 1 ? 3 : 2) void k_pool_attn(AttnArgs a) {
  constexpr int NC = (HD + 63) / 64;            // 64-column chunks of a K row
  constexpr int NV = (HD / 16 + 3) / kWaves;    // 16-column tiles of V for a wave
  __shared__ int4 sp[kWaves][RT][2][2][64];     // the weights' pieces, eight tokens each
  __shared__ __align__(16) _Float16 sq[2][16 * RT][NC * 64 + 8];  // the rows' pieces
  __shared__ float sqs[16 * RT];                   // and what they are multiplied by
  __shared__ int spg[kPages];
  __shared__ float smax[kWaves][RT][16], smaxs[kWaves][RT][16];
  __shared__ float ssum[kWaves][RT][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  int slot, z;
  work_of(a, &slot, &z);
  const int hy = blockIdx.y;
  const int kvh = hy / a.hgroups, hg = hy % a.hgroups;
  SeqRows seq;
  Tile t = tile_of(a, slot, &seq);
  if (t.queries == 0) {
    if (a.splits > 1 && z == 0 && hy == 0 && threadIdx.x == 0) a.meta[slot] = make_int4(0, 0, 0, 0);
    return;
  }
  // What hangs on the sequence alone is fetched together: the first round's pages where no window
  // moves it (one of its 16 blocks in each lane group's lanes; -1: none), q, the length.
  // Pages stand for the first of this kv head's blocks in them: below 2^31 in a layer.
  const int pshift = a.p.page_shift - 4, pmask = (1 << pshift) - 1;
  auto page_of = [&](int T0) {
    const int g = page_at(a.p, t.seq, T0 >> a.p.page_shift);
    return g < 0 ? -1 : (g * a.p.n_kv_heads + kvh) << pshift;
  };
  auto pages = [&](int T0) { return page_of(T0 + 16 * n); };
  int pg = -1;
  if (a.window == 0) pg = pages(z * a.chunk);
  // q: kPer lanes share a row, four columns each; a wave takes every fourth set of rows.
  constexpr int kPer = NC == 1 ? 16 : NC == 2 ? 32 : 64, kSets = 64 / kPer;
  constexpr int kTurns = 16 * RT / (kWaves * kSets);
  const int qc = lane % kPer * 4;
  float4 x[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; i++) {
    const int at = (i * kWaves + wave) * kSets + lane / kPer;
    const int qi = at / a.hpt, hh = hg * a.hpt + at % a.hpt;
    x[i] = make_float4(0, 0, 0, 0);
    if (qi < t.queries && hh < a.group && qc < HD)
      x[i] = *reinterpret_cast<const float4*>(a.q + (t.row0 + qi) * a.q_stride +
                                              (long)(kvh * a.group + hh) * HD + qc);
  }
  tile_len(a, seq, &t);
  int lo, hi, tb, te;
  tile_range(a, t, &lo, &hi);
  part_range(a, lo, hi, z, &tb, &te);
  if (a.splits > 1 && z == 0 && hy == 0 && threadIdx.x == 0)  // for the joining launch
    a.meta[slot] = make_int4(t.row0, t.queries, hi > lo ? (hi - lo - 1) / a.chunk + 1 : 0, 0);
  if (tb >= te && a.splits > 1) return;
  if (a.window > 0) pg = pages(tb);
  if (tb + 16 * n >= te) pg = -1;
  // Those of later rounds by way of LDS, kPages blocks at a time: a load of them in the
  // loop would wait for the V before it.
  auto fill_pages = [&](int T0) {
    for (int i = threadIdx.x; i < kPages && T0 + 16 * i < te; i += 256)
      spg[i] = page_of(T0 + 16 * i);
  };
  const bool more = tb + kRound < te;
  if (more) fill_pages(tb);
  const int8_t* const data = a.p.data;

  // this lane's rows
  long row[RT];
  int head[RT], row_hi[RT], row_lo[RT];
  bool row_ok[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const int at = 16 * r + n, qi = at / a.hpt, hh = hg * a.hpt + at % a.hpt;
    row_ok[r] = qi < t.queries && hh < a.group;
    // a lane without a row computes row 0 again and writes nothing
    row[r] = t.row0 + (row_ok[r] ? qi : 0);
    head[r] = kvh * a.group + (row_ok[r] ? hh : hg * a.hpt);
    // positions before 0 see nothing
    row_hi[r] = row_ok[r] && t.pos0 + qi >= 0 ? t.pos0 + qi + 1 : 0;
    row_lo[r] = a.window > 0 ? row_hi[r] - a.window : 0;
  }

  // K of the wave's step, its blocks' scales, and V's columns of the round
  int4 kr[4][NC], vr[NV][kWaves];
  float2 sc;
  bool here;
  const int kb = 4 * wave + (n >> 2);  // the round's block of the lane's K rows
  int kp = -1, wp = -1, vp[kWaves];  // pages of its K, its scales, and V's four blocks
  // What is not there: the first page's.
  auto block = [&](int page, int b) { return (uint32_t)((page < 0 ? 0 : page) + (b & pmask)); };
  auto load_k = [&](int T0) {
    const int b0 = T0 >> 4;
    const int8_t* s = data + (size_t)block(kp, b0 + kb) * (2 * kKvBlock * HD) + (n & 3) * HD +
                      (16 * g < HD ? 16 * g : 0);
#pragma unroll
    for (int tt = 0; tt < 4; tt++)
#pragma unroll
      for (int c = 0; c < NC; c++)
        // columns behind the row: the lane's first ones again, against a q of 0
        kr[tt][c] = load16(s + 4 * tt * HD + (HD % 64 == 0 || 64 * c + 16 * g < HD ? 64 * c : 0));
    here = wp >= 0;
    sc = make_float2(0.0f, 0.0f);
    if (here)
      sc = reinterpret_cast<const float2*>(a.p.scale)[block(wp, b0 + 4 * wave + g)];
  };
  // A tile behind the last is an earlier one again and never stored: a branch around it in the
  // loop cost head_dim 96 18 spilled registers (4 x 1000 tokens 18.9 us, 14.3 without) and
  // 224 its second workgroup (32 x 1500: 26.9 us, 17.1).
  int vtile[NV];
#pragma unroll
  for (int d = 0; d < NV; d++)
    vtile[d] = HD % 64 == 0 || wave + 4 * d < HD / 16 ? wave + 4 * d : wave % (HD / 16);
  auto load_v = [&](int T0) {
#pragma unroll
    for (int s = 0; s < kWaves; s++) {
      const int8_t* v = data + (size_t)block(vp[s], (T0 >> 4) + 4 * s + g) * (2 * kKvBlock * HD) +
                        kKvBlock * HD + n * kKvBlock;
#pragma unroll
      for (int d = 0; d < NV; d++)
        vr[d][s] = load16(v + vtile[d] * 16 * kKvBlock);
    }
  };
  if (tb < te) {
    kp = __shfl(pg, kb);
    wp = __shfl(pg, 4 * wave + g);
#pragma unroll
    for (int s = 0; s < kWaves; s++) vp[s] = __shfl(pg, 4 * s + g);
    load_k(tb);
  }

  // q's pieces, for all waves: times a power of two that brings the row's largest to 2^14 .. 2^15
#pragma unroll
  for (int i = 0; i < kTurns; i++) {
    const int at = (i * kWaves + wave) * kSets + lane / kPer;
    const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float amax = 0.0f, bad = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float f = fabsf(v[j]);
      amax = fmaxf(amax, f);
      bad = f <= 3.402823466e+38f ? bad : 1.0f;
    }
    amax = row_max(amax);
    bad = row_max(bad);
    if (kPer >= 32) {
      amax = fmaxf(amax, lane_xor_f<16>(amax));
      bad = fmaxf(bad, lane_xor_f<16>(bad));
    }
    if (kPer == 64) {
      amax = fmaxf(amax, lane_xor_f<32>(amax));
      bad = fmaxf(bad, lane_xor_f<32>(bad));
    }
    // (a row below 2^-96 less far: the factor that takes it back stays a normal number)
    const int e = 15 - __builtin_amdgcn_frexp_expf(amax), up = e < 111 ? e : 111;
    int2 p0, p1;
    pieces2(__builtin_ldexpf(v[0], up), __builtin_ldexpf(v[1], up), &p0.x, &p1.x);
    pieces2(__builtin_ldexpf(v[2], up), __builtin_ldexpf(v[3], up), &p0.y, &p1.y);
    if (qc < NC * 64) {
      *reinterpret_cast<int2*>(&sq[0][at][qc]) = p0;
      *reinterpret_cast<int2*>(&sq[1][at][qc]) = p1;
    }
    if (qc == 0) sqs[at] = bad > 0.0f ? NAN : __builtin_ldexpf(a.scale2, -up);
  }
  __syncthreads();
  float qs[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) qs[r] = sqs[16 * r + n];

  float o[RT][NV][4], M[RT], N[RT], L[RT];
  float top[RT], tops[RT];  // the largest weight's power so far, and the largest score's
#pragma unroll
  for (int r = 0; r < RT; r++) {
    M[r] = N[r] = top[r] = tops[r] = kNone;
    L[r] = 0.0f;
#pragma unroll
    for (int d = 0; d < NV; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[r][d][i] = 0.0f;
  }

  for (int T0 = tb; T0 < te; T0 += kRound) {
    const int Tw = T0 + wave * kStep;  // of the wave
    const bool mine = Tw < te;
    float e[RT][16], mx[RT];  // exponents, and their largest of the lane's block
    float evf = 0.0f, fw = 0.0f, lf = 0.0f;
#pragma unroll
    for (int r = 0; r < RT; r++) mx[r] = kNone;
    if (mine) {
      __builtin_amdgcn_s_setprio(1);
      // Exponents: scores in powers of two, with V's.
      const float vs = sc.y;
      int ev = kMinExp;
      float f = vs * 0x1p125f;
      if (vs >= 0x1p-126f) {
        ev = __builtin_amdgcn_frexp_expf(vs);
        f = __builtin_amdgcn_frexp_mantf(vs);
      }
      fw = f * kTop;
      lf = fmaxf(__builtin_amdgcn_logf(f), -1.0f);
      evf = (float)ev;
      // Every token of the step seen by every row of the tile?
      const bool full = __all(here) && Tw + kStep <= t.pos0 + 1 &&
                        (a.window == 0 || Tw >= t.pos0 + t.queries - a.window);
      v8h qd[RT][NC][2][2];
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 2; i++)
              qd[r][k][h][i] =
                  *reinterpret_cast<const v8h*>(&sq[i][16 * r + n][64 * k + 16 * g + 8 * h]);
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
        v4f acc[RT][2];
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r][0] = acc[r][1] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const v8h kk = h ? widened(kr[tt][k].z, kr[tt][k].w) : widened(kr[tt][k].x, kr[tt][k].y);
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
              for (int i = 0; i < 2; i++) acc[r][i] = mfma(kk, qd[r][k][h][i], acc[r][i]);
          }
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            e[r][4 * tt + i] = __builtin_fmaf(
                __builtin_fmaf(acc[r][1][i], 1.0f / kSecond, acc[r][0][i]), qs[r] * sc.x, evf);
      }
#pragma unroll
      for (int r = 0; r < RT; r++) {
        if (!full) {
          const int first = row_lo[r] - (Tw + 16 * g);
          const unsigned seen = here ? row_hi[r] - row_lo[r] : 0;
#pragma unroll
          for (int j = 0; j < 16; j++) e[r][j] = (unsigned)(j - first) < seen ? e[r][j] : kNone;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) mx[r] = fmaxf(mx[r], e[r][j]);
      }
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      // Powers so large that f (V's exponent) is within their rounding: without it, which errs to
      // the safe side (and for N, any number near the scores' largest will do).
      const float x = fabsf(mx[r]);
      const float m = rows_larger(x < kLarge ? mx[r] + lf : mx[r]);
      const float s = rows_larger(x < 0x1p24f ? mx[r] - evf : mx[r]);
      if (g == 0) {
        smax[wave][r][n] = m;
        smaxs[wave][r][n] = s;
      }
    }
    __builtin_amdgcn_s_setprio(0);
    // This round's V, and behind it the next one's K.
    load_v(T0);
    const int Tn = T0 + kRound;
    if (Tn < te) {
      const int at = (Tn - tb) >> 4 & (kPages - 1);
      if (at == 0) {
        __syncthreads();
        fill_pages(Tn);
        __syncthreads();
      }
      const int left = (te - Tn + 15) >> 4;  // blocks
      kp = kb < left ? spg[at + kb] : -1;
      wp = 4 * wave + g < left ? spg[at + 4 * wave + g] : -1;
#pragma unroll
      for (int s = 0; s < kWaves; s++) vp[s] = 4 * s + g < left ? spg[at + 4 * s + g] : -1;
      load_k(Tn);
    }
    __syncthreads();
    float alpha[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const float round = larger(larger(larger(smax[0][r][n], smax[1][r][n]), smax[2][r][n]),
                                 smax[3][r][n]);
      top[r] = larger(top[r], round);
      const float to = reference(larger(round, top[r] - kFall));
      // (of the maximum, never of the N before: a reference's own reference lies above it, and a
      // denominator against what rises every round vanishes after 2000 of them)
      tops[r] = larger(larger(larger(larger(tops[r], smaxs[0][r][n]), smaxs[1][r][n]), smaxs[2][r][n]),
                       smaxs[3][r][n]);
      const float tos = reference(tops[r]);
      const float ref = to == kNone ? 0.0f : to, refs = tos == kNone ? 0.0f : tos;
      alpha[r] = lift(M[r], ref);
      L[r] *= lift(N[r], refs);
      M[r] = to;
      N[r] = tos;
      if (mine) {
        // 0 but for blocks far below M (and 300 for those that nothing is seen of)
        const float deep = fminf(fmaxf(ceilf(ref - mx[r]) - kDeep, 0.0f), 300.0f);
        const float base = ref - deep, down = ref - base;
        const float fwd = __builtin_ldexpf(fw, -(int)down);
        float sum = 0.0f;
        int4 p[2][2];
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = __builtin_amdgcn_exp2f(e[r][4 * tt + i] - base);
            sum += x;
            w[i] = x * fwd;
          }
          const int at = 2 * (tt & 1), h = tt >> 1;
          pieces2(w[0], w[1], &p[0][h].x + at, &p[1][h].x + at);
          pieces2(w[2], w[3], &p[0][h].x + at + 1, &p[1][h].x + at + 1);
        }
        L[r] = __builtin_fmaf(sum, __builtin_amdgcn_exp2f((ref - refs) - down - evf), L[r]);
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) sp[wave][r][k][h][lane] = p[k][h];
      } else {
        // no tokens: weights of 0, whatever V holds there
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) sp[wave][r][k][h][lane] = make_int4(0, 0, 0, 0);
      }
    }
    __syncthreads();
    __builtin_amdgcn_s_setprio(1);
    // Values of 256 tokens, each piece's apart; in two chains where there is one tile.
    constexpr int kChains = RT * NV < 2 ? 2 : 1;
    v4f acc[RT][NV][kChains][2];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int d = 0; d < NV; d++)
#pragma unroll
        for (int j = 0; j < kChains; j++) acc[r][d][j][0] = acc[r][d][j][1] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < kWaves; s++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int j = h % kChains;
        v8h w[RT][2];
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int k = 0; k < 2; k++) w[r][k] = __builtin_bit_cast(v8h, sp[s][r][k][h][lane]);
#pragma unroll
        for (int d = 0; d < NV; d++) {
          const v8h v = h ? widened(vr[d][s].z, vr[d][s].w) : widened(vr[d][s].x, vr[d][s].y);
#pragma unroll
          for (int r = 0; r < RT; r++)
#pragma unroll
            for (int k = 0; k < 2; k++) acc[r][d][j][k] = mfma(v, w[r][k], acc[r][d][j][k]);
        }
      }
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int d = 0; d < NV; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float hi = acc[r][d][0][0][i], lo = acc[r][d][0][1][i];
          if (kChains == 2) {
            hi += acc[r][d][kChains - 1][0][i];
            lo += acc[r][d][kChains - 1][1][i];
          }
          o[r][d][i] = __builtin_fmaf(o[r][d][i], alpha[r], __builtin_fmaf(lo, 1.0f / kSecond, hi));
        }
    __builtin_amdgcn_s_setprio(0);
  }

  // The waves' denominators; then each wave has its columns' results.
#pragma unroll
  for (int r = 0; r < RT; r++) {
    L[r] = rows_sum(L[r]);
    if (g == 0) ssum[wave][r][n] = L[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; r++) {
    if (!row_ok[r]) continue;
    const float l = (ssum[0][r][n] + ssum[1][r][n]) + (ssum[2][r][n] + ssum[3][r][n]);
    if (a.splits == 1) {
      const Over over(M[r], N[r], l);
      float* dst = a.out + row[r] * a.out_stride + (long)head[r] * HD + 4 * g;
#pragma unroll
      for (int d = 0; d < NV; d++)
        if (HD % 64 == 0 || wave + 4 * d < HD / 16)
          *reinterpret_cast<float4*>(dst + 16 * (wave + 4 * d)) = make_float4(
              over(o[r][d][0]), over(o[r][d][1]), over(o[r][d][2]), over(o[r][d][3]));
    } else {
      const size_t at =
          ((size_t)(slot * gridDim.y + hy) * a.splits + z) * (16 * RT) + 16 * r + n;
#pragma unroll
      for (int d = 0; d < NV; d++)
        if (HD % 64 == 0 || wave + 4 * d < HD / 16)
          *reinterpret_cast<float4*>(a.part + at * HD + 16 * (wave + 4 * d) + 4 * g) =
              make_float4(o[r][d][0], o[r][d][1], o[r][d][2], o[r][d][3]);
      if (wave == 0 && g == 0)
        *reinterpret_cast<float4*>(a.ml + 4 * at) = make_float4(M[r], N[r], l, 0.0f);
    }
  }
}

// The parts of each row joined, by W waves a row: one where parts are few (a
// workgroup then joins four rows), four where one wave would be left with long loops.  The
// loads are of addresses that the grid alone gives, all at once: the first part's
// workgroup left the tile's rows and number of parts.
template <int HD, int W>
__global__ __launch_bounds__(256) void k_pool_attn_join(AttnArgs a) {
  constexpr int Q = HD / 4, G = 64 * W / Q;  // threads of a part's columns, parts side by side
  constexpr int kEach = W == 1 ? 1 : kMaxParts / 256, kAhead = W == 1 ? 8 : 4;
  __shared__ float weight[W == 1 ? 1 : kMaxParts];
  __shared__ float red[12];
  __shared__ __align__(16) float sums[W == 1 ? 1 : G][HD];
  const int rows = 16 * a.rt, tid = threadIdx.x % (64 * W);
  const int item = blockIdx.x * (4 / W) + threadIdx.x / (64 * W);
  const int n = item % rows, slot = item / rows, hy = blockIdx.y;
  const size_t at = (size_t)(slot * gridDim.y + hy) * a.splits * rows + n;
  const int4 meta = a.meta[slot];
  float m[kEach], ns[kEach], l[kEach];
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int s = tid + 256 * j;
    float4 v = make_float4(kNone, kNone, 0.0f, 0.0f);
    if (s < a.splits) v = *reinterpret_cast<const float4*>(a.ml + 4 * (at + (size_t)s * rows));
    m[j] = v.x;
    ns[j] = v.y;
    l[j] = v.z;
  }
  const int c = tid % Q, grp = tid / Q;
  const float* part = a.part + at * HD + 4 * c;
  float4 v[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; j++) {
    const int s = grp + j * G;
    v[j] = make_float4(0, 0, 0, 0);
    if (grp < G && s < a.splits)
      v[j] = *reinterpret_cast<const float4*>(part + (size_t)s * rows * HD);
  }
  const int qi = n / a.hpt, hh = hy % a.hgroups * a.hpt + n % a.hpt;
  if (!(qi < meta.y && hh < a.group)) return;
  const int parts = meta.z < a.splits ? meta.z : a.splits;
  float M = kNone, N = kNone, L = 0.0f;
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    if (tid + 256 * j >= parts) {  // a part that is not there holds anything
      m[j] = ns[j] = kNone;
      l[j] = 0.0f;
    }
    M = fmaxf(M, m[j]);
    N = fmaxf(N, ns[j]);
  }
  M = wave_max(M);
  N = wave_max(N);
  if (W > 1) {
    if ((tid & 63) == 0) {
      red[tid >> 6] = M;
      red[8 + (tid >> 6)] = N;
    }
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    N = fmaxf(fmaxf(red[8], red[9]), fmaxf(red[10], red[11]));
  }
  const float ref = M == kNone ? 0.0f : M, refs = N == kNone ? 0.0f : N;
  float w[kEach];
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    w[j] = lift(m[j], ref);
    if (W > 1) weight[tid + 256 * j] = w[j];
    L += lift(ns[j], refs) * l[j];
  }
  L = wave_sum(L);
  if (W > 1) {
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = L;
    __syncthreads();
    L = (red[4] + red[5]) + (red[6] + red[7]);
  }
  float4 o = make_float4(0, 0, 0, 0);
  for (int s0 = 0; s0 < parts; s0 += kAhead * G) {
    float4 u[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int s = s0 + grp + (kAhead + j) * G;
      u[j] = make_float4(0, 0, 0, 0);
      if (grp < G && s < parts)
        u[j] = *reinterpret_cast<const float4*>(part + (size_t)s * rows * HD);
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int s = s0 + grp + j * G;
      const float f = W > 1 ? weight[s < kMaxParts ? s : 0] : __shfl(w[0], s & 63);
      if (s < parts) {
        o.x += f * v[j].x;
        o.y += f * v[j].y;
        o.z += f * v[j].z;
        o.w += f * v[j].w;
      }
      v[j] = u[j];
    }
  }
  float* dst = a.out + (long)(meta.x + qi) * a.out_stride + (long)(hy / a.hgroups * a.group + hh) * HD;
  const Over over(M, N, L);
  if (W == 1) {
    float4 r = o;
#pragma unroll
    for (int j = 1; j < G; j++) {
      r.x += __shfl(o.x, tid + j * Q);
      r.y += __shfl(o.y, tid + j * Q);
      r.z += __shfl(o.z, tid + j * Q);
      r.w += __shfl(o.w, tid + j * Q);
    }
    if (tid < Q)
      *reinterpret_cast<float4*>(dst + 4 * c) =
          make_float4(over(r.x), over(r.y), over(r.z), over(r.w));
  } else {
    if (grp < G) *reinterpret_cast<float4*>(&sums[grp][4 * c]) = o;
    __syncthreads();
    if (tid < HD) {
      float sum = 0.0f;
      for (int j = 0; j < G; j++) sum += sums[j][tid];
      dst[tid] = over(sum);
    }
  }
}

// How the work is cut.  Heads: at most 16 of a kv head's query heads share a
// tile, as many queries beside each other as fill it; 32 rows where sequences bring
// as many.  Tokens: a tile's part is one workgroup.  The number of rounds of a part is the
// one with the least time by what was measured (us): 4.5 before a workgroup's first
// round and after its last, 0.7 + 0.014 head_dim a round, 5 for a thousand workgroups, 4 for
// joining parts; 768 workgroups at once (512 where registers allow two a CU), of
// several sequences 0.6 of the longest's parts filled.  (702 tokens of head_dim 64: one part
// 9.2, three 9.6; 1500 of 128: one 19.7, six 11.3; 16 sequences of up to 1024: one 15.0, four
// 12.1; 64 of them: one 17.2, four 19.3; 32 of up to 4096: eight 23.8, four 24.3, sixteen 27.9;
// 8 of up to 2000 of head_dim 256: eight 14.2, four 18.5.)
AttnArgs attn_plan(const PoolView& p, const Ragged& r, int n_heads, int max_len, int window) {
  AttnArgs a = {};
  a.p = p;
  a.r = r;
  a.group = n_heads / p.n_kv_heads;
  a.hgroups = (a.group + 15) / 16;
  a.hpt = (a.group + a.hgroups - 1) / a.hgroups;
  a.rt = p.hd <= 128 && (long)r.T * a.hpt >= 32l * r.n ? 2 : 1;
  a.qpt = 16 * a.rt / a.hpt;
  a.extra = 1;
  if (r.T <= r.n) {  // one row a sequence: a tile for each row, and no slot to spare
    a.qpt = 1;
    a.extra = 0;
  }
  a.window = window;
  a.slots = r.T / a.qpt + a.extra * r.n;
  long range = max_len;
  if (window > 0 && window + (long)a.qpt + kStep < range) range = window + (long)a.qpt + kStep;
  const long y = (long)p.n_kv_heads * a.hgroups;
  const long tiles = (r.T / a.qpt > r.n ? r.T / a.qpt : r.n) * y;
  const float at_once = a.rt == 1 && p.hd <= 128 ? 768.0f : 512.0f, filled = r.n > 1 ? 0.6f : 1.0f;
  const long most = (range + kRound - 1) / kRound;
  float best = INFINITY;
  long chunk = 0;
  for (long rounds = 1;; rounds += 1 + rounds / 4) {
    if (rounds > most) rounds = most;
    const long parts = (most + rounds - 1) / rounds;
    if (parts == 1 || (parts <= kMaxParts && parts * a.slots * y <= kMostItems)) {
      const float wgs = (float)tiles * (float)parts;
      const float turns = parts > 1 ? wgs * filled / at_once : wgs / at_once;
      const float us = (turns > 1.0f ? turns : 1.0f) *
                           (4.5f + (0.7f + 0.014f * (float)p.hd) * (float)rounds) +
                       0.005f * wgs + (parts > 1 ? 4.0f : 0.0f);
      if (us < best) {
        best = us;
        chunk = rounds * kRound;
      }
    }
    if (rounds == most) break;
  }
  a.chunk = (int)chunk;
  a.splits = (int)((range + chunk - 1) / chunk);
  return a;
}

// Rows of all parts.
size_t part_rows(const AttnArgs& a) {
  return (size_t)a.slots * a.p.n_kv_heads * a.hgroups * a.splits * (16 * a.rt);
}

template <int HD>
void attn_launch(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.slots * a.splits), (unsigned)(a.p.n_kv_heads * a.hgroups));
  if (a.rt == 1) hipLaunchKernelGGL((k_pool_attn<HD, 1>), grid, dim3(256), 0, st, a);
  if constexpr (HD <= 128)
    if (a.rt == 2) hipLaunchKernelGGL((k_pool_attn<HD, 2>), grid, dim3(256), 0, st, a);
  if (a.splits > kJoinWave)
    hipLaunchKernelGGL((k_pool_attn_join<HD, 4>), dim3(16 * a.rt * a.slots, grid.y), dim3(256), 0,
                       st, a);
  else if (a.splits > 1)
    hipLaunchKernelGGL((k_pool_attn_join<HD, 1>), dim3(4 * a.rt * a.slots, grid.y), dim3(256), 0,
                       st, a);
}

}  // namespace

size_t kv_attention_scratch(const PoolView& p, const Ragged& r, int n_heads, int max_len,
                            int window) {
  const AttnArgs a = attn_plan(p, r, n_heads, max_len, window);
  return a.splits == 1 ? 0 : part_rows(a) * (p.hd + 4) * sizeof(float) + a.slots * sizeof(int4);
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
  a.ml = a.part + part_rows(a) * p.hd;
  a.meta = reinterpret_cast<int4*>(a.ml + part_rows(a) * 4);
  switch (p.hd) {
    case 32: attn_launch<32>(a, st); break;
    case 64: attn_launch<64>(a, st); break;
    case 96: attn_launch<96>(a, st); break;
    case 128: attn_launch<128>(a, st); break;
    case 160: attn_launch<160>(a, st); break;
    case 192: attn_launch<192>(a, st); break;
    case 224: attn_launch<224>(a, st); break;
    default: attn_launch<256>(a, st); break;
  }
  return hipGetLastError();
}

}  // namespace qr
