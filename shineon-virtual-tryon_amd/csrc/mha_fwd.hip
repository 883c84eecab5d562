// Multi-head attention with a learned relative position bias, forward, gfx950.
//
//   o_i = sum_j softmax_j(scale q_i . k_j + bias_h[code_j - code_i]) v_j,   j over the visible keys; a row without any gives 0
//
// One pass over the keys per row of queries: running maximum m, running sum l and o unnormalised in registers (fp32), rescaled when m
// moves.  The bias is the learned table expanded over offsets (so_mha_prep: one float per head and offset, divided by scale) and
// ENTERS AS THE INITIAL ACCUMULATOR of the q k^T product, so adding it costs no vector instruction beyond its load: the scores in
// log2 units are acc * (scale log2 e) in one multiply-add with -m.
//
// A block is four waves; mha_fwd_k takes 128 rows of a head, mha_few_k (at most 32 rows to a key head) all rows and cuts the keys over its
// waves.  When there are too few blocks to fill the chip the keys are cut into parts as well, each leaves (o, m, l) in fp32 and mha_join_k
// merges them.
#include <math.h>
#include "mha.h"

using namespace mha;

namespace {

struct FwdP {
  so_mha_desc d;
  int parts, row_tiles;
  int stages, stage_bytes, seg;      // seg: floats of the bias that a tile of 64 and a block of 128 tokens can meet, in whole 64s
  float c;              // scale * log2 e
};

constexpr int kLds = 160 * 1024;

// A row's softmax for the backward pass: reference and 1 / l apart.  Their sum in log2 units would lose l where scores are large (at 2^30 a
// step of fp32 is 64 to 128), and with it the rounding of m, which is a common factor of the row's probabilities that l carries too.
__device__ __forceinline__ void write_stats(const so_mha_desc& D, int b, int head, int qi, float m, float l, float inv) {
  const size_t at = ((size_t)b * D.Hq + head) * D.Lq + qi;
  D.stats[at] = l == 0.f ? INFINITY : m;
  D.stats[(size_t)D.B * D.Hq * D.Lq + at] = inv;
}

// one row's result: o / l (or o, m, l of a part) and its statistics
template <typename T, int NT>
__device__ __forceinline__ void write_row(const FwdP& P, const f32x16 (&o)[NT], float m, float l, int b, int hk, int head, int qi, int part, int half) {
  const so_mha_desc& D = P.d;
  if (P.parts > 1) {      // unnormalised rows and statistics for mha_join_k: [b][Hk][rows][parts]
    const int G = D.Hq / D.Hk;
    const size_t at = (((size_t)b * D.Hk + hk) * G * D.Lq + (size_t)(head - hk * G) * D.Lq + qi) * P.parts + part;
    if (half == 0) {
      D.part_ml[2 * at] = m;
      D.part_ml[2 * at + 1] = l;
    }
    float* po = D.part_o + at * D.D;
#pragma unroll
    for (int v = 0; v < NT; ++v)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * v + 8 * g + 4 * half;
        if (c < D.D) *reinterpret_cast<f32x4*>(po + c) = f32x4{o[v][4 * g], o[v][4 * g + 1], o[v][4 * g + 2], o[v][4 * g + 3]};
      }
    return;
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;        // an empty row gives zeros, NaN stays NaN
  const size_t orow = ((size_t)b * D.Lq + qi) * D.Hq + head;
  T* op = (T*)D.o + orow * D.D;
  float* fp = D.o_f32 ? D.o_f32 + orow * D.D : nullptr;
#pragma unroll
  for (int v = 0; v < NT; ++v)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * v + 8 * g + 4 * half;
      if (c < D.D) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        f32x4 x;
        t4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = o[v][4 * g + e] * inv;
          y[e] = (T)x[e];
        }
        *reinterpret_cast<t4*>(op + c) = y;
        if (fp) *reinterpret_cast<f32x4*>(fp + c) = x;
      }
    }
  if (D.stats && half == 0) write_stats(D, b, head, qi, m, l, inv);
}

// The running softmax of 32 keys per half: s -> probabilities against the reference m; o and l are rescaled when m moves.  m follows the
// maximum only when that has grown by more than kSlack (log2 units): probabilities up to 2^kSlack lose nothing in a floating-point type,
// and after a row's first tiles hardly any tile rescales (following every growth: 380 instead of 366 us at 8191 tokens, 16 heads of 64,
// with probabilities in one piece).
constexpr float kSlack = 8.f;
template <int N, int NT>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[N], f32x16 (&o)[NT], float& m, float& l, float c) {
  float mx = -INFINITY;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
  mx = half_max(mx) * c;
  if (__any(mx > m + kSlack)) {
    const float mn = fmaxf(m, mx), alpha = exp2_(m - (mn == -INFINITY ? 0.f : mn));
    m = mn;
    l *= alpha;
#pragma unroll
    for (int v = 0; v < NT; ++v)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[v][r] *= alpha;
  }
  const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[u][r] = exp2_(__builtin_fmaf(s[u][r], c, -ms));
      l += s[u][r];
    }
}

// Probabilities as operands of the product with v.  bf16: in three pieces, each the 8 bits of what the ones before leave, multiplied one after
// the other, so that all 24 bits take part.  One piece adds as much error to o as o's own rounding (2.3e-3 instead of 1.7e-3 of its norm), two
// show in delta = do . o against the probabilities that the backward pass rebuilds: the bias gradient's sums over rows cancel, and it is 2 to
// 5 times further off.  Pieces by what wants a gradient would make o's bits depend on that.  (8191 tokens, 16 heads of 64: 354-360, 487,
// 596-616 us with one, two, three.)
template <typename T> constexpr int kPieces = sizeof(T) == 2 ? 3 : 1;
template <typename T, int NCS>
__device__ __forceinline__ void prob_frags(const f32x16& s, typename Elem<T>::frag (&p)[kPieces<T>][NCS]) {
  constexpr int E = Elem<T>::E;
#pragma unroll
  for (int c = 0; c < NCS; ++c) {
    to_frag(s, c, p[0][c]);
    f32x16 rest;
#pragma unroll
    for (int i = 1; i < kPieces<T>; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) rest[E * c + e] = (i == 1 ? s : rest)[E * c + e] - (float)p[i - 1][c][e];
      to_frag(rest, c, p[i][c]);
    }
  }
}

// Many rows: a block is 128 rows of one head, 32 per wave, and walks 64-key tiles.  BIAS: 0 none, 1 sequence, 2 map; the piece of the
// expanded bias that a tile's offsets lie in travels to LDS with the tile.  (Read from global memory by every lane it took 120 of 495 us
// at 8191 tokens, 16 heads of 64.)
//
// fp32 is bound by the matrix pipes (80 % busy: 287 us, 120 TFLOP/s at 4 x 2048 tokens, 8 heads of 64).  bf16, four products for the formula's
// two, by matrix and vector instructions one after the other: at 128 channels 51 and at least 46 % of the SIMD cycles (2 x 4097 tokens, 16 heads:
// 604 us, 910 TFLOP/s of executed products), at 64 channels 42 and 67 % (8191 tokens, 16 heads: 596-690 us, 800-920 TFLOP/s).
// (Two waves per SIMD in fp32 end at 64 channels: at 96 their registers spill, 4 x 2048 tokens, 8 heads 490 against 455 us.)
template <typename T, int DP, int BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? (DP <= 64 ? 3 : 2) : (DP <= 64 ? 2 : 1))) void mha_fwd_k(const FwdP P) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::frag frag;
  constexpr int E = Elem<T>::E, KM = 2 * E, NM = DP / KM, NT = DP / 32, NCS = 32 / KM;
  constexpr int TK = 64, TILE = TK * TL::kRowBytes, HALF = TILE / 2;
  extern __shared__ __attribute__((aligned(512))) char sm[];         // [stages][K tile | V tile | bias | codes]
  const so_mha_desc& D = P.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, half = lane >> 5;
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const int G = D.Hq / D.Hk;
  const BlockOf blk = block_of(D.B, D.Hk, G * P.row_tiles * P.parts);
  const int b = blk.b, hk = blk.hk, part = blk.idx / (G * P.row_tiles), gt = blk.idx - part * G * P.row_tiles;
  const int head = hk * G + gt / P.row_tiles, q0 = gt % P.row_tiles * 128;
  const int qlast = (q0 + 128 < D.Lq ? q0 + 128 : D.Lq) - 1, row = q0 + 32 * wave + li;
  const bool rowv = row < D.Lq;
  const int qi = rowv ? row : qlast;
  const bool idle = !__any(rowv);      // this wave only helps to fill tiles

  const unsigned long long* words = D.words ? (const unsigned long long*)D.words + (size_t)b * D.nwords : nullptr;
  int t0, t1;
  word_range(words, D.Lk, lane, t0, t1);
  if (P.parts > 1) {
    const int n = t1 > t0 ? t1 - t0 : 0, per = (n + P.parts - 1) / P.parts;
    t0 += part * per;
    t1 = t0 + per < t1 ? t0 + per : t1;
  }

  frag q[NM];
  {
    const T* qr = (const T*)D.q + (size_t)b * D.sqb + (size_t)qi * D.sql + (size_t)head * D.sqh;
#pragma unroll
    for (int m = 0; m < NM; ++m) q[m] = as_frag<T>(load_chunk<T>(qr, 2 * m + half, rowv && (2 * m + half) * E < D.D));
  }
  // first offset of tile t's piece of the bias: code(first key) - code(last row); this lane's place in it
  const int STAGE = P.stage_bytes;
  const int cqf = BIAS == 2 ? D.code[D.q_start + q0] : 0;
  const int cqe = BIAS == 0 ? 0 : BIAS == 1 ? D.q_start + q0 + 127 : D.code[D.q_start + qlast];
  const int mine_q = BIAS == 0 ? 0 : BIAS == 1 ? 127 - 32 * wave - li + 16 * half : cqe - D.code[D.q_start + qi];
  const float* bias = BIAS ? D.bias + (size_t)head * D.V + D.code_max - cqe : nullptr;

  const T* kb = (const T*)D.k + (size_t)b * D.skb + (size_t)hk * D.skh;
  const T* vb = (const T*)D.v + (size_t)b * D.svb + (size_t)hk * D.svh;
  const Filler<T, DP, TK, 4> fk(D.D, (unsigned)(D.skl * sizeof(T)), tid), fv(D.D, (unsigned)(D.svl * sizeof(T)), tid);
  const Reader<T, DP> rd(sm, lane);
  KeyWords kw(words, D.nwords, D.Lk, lane);
  unsigned long long next = 0;
  auto fetch = [&](int t, int st) {
    next = kw.get(t);
    char* kt = sm + st * STAGE;
    fk.fill(kt, kb + (size_t)t * TK * D.skl, next, 0, wave_u);
    fv.fill(kt + TILE, vb + (size_t)t * TK * D.svl, next, 0, wave_u);
    if constexpr (BIAS == 1) fill_dwords<4>(kt + 2 * TILE, bias + t * TK, TK + 127, 0x7FFFFFFFu, wave_u, lane);
    if constexpr (BIAS == 2) {
      const int c0 = D.code[t * TK];
      fill_dwords<4>(kt + 2 * TILE, bias + c0, D.code[t * TK + TK - 1] - cqf - (c0 - cqe) + 1, 0x7FFFFFFFu, wave_u, lane);
      fill_dwords<4>(kt + 2 * TILE + 4 * P.seg, D.code + t * TK, TK, 0x7FFFFFFFu, (wave_u + 1) & 3, lane);
    }
  };

  frag f[NM];      // NM = NT * NCS: every phase has as many steps
  f32x16 o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (t0 < t1) fetch(t0, 0);
#pragma unroll
  for (int m = 0; m < NM; ++m) settle(q[m]);
  drain();
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int st = P.stages == 2 ? (t - t0) & 1 : 0;
    const int fr = rd.rows + st * STAGE, fc = rd.cols + st * STAGE;
    const int seg = opaque(lds_at(sm) + st * STAGE + 2 * TILE + 4 * mine_q);      // this lane's place in the tile's piece of the bias
    const unsigned long long w64 = next;
    if (P.stages == 2 && t + 1 < t1) fetch(t + 1, st ^ 1);
    if (!idle) {
    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (BIAS == 1) {
        lds_read16(seg + 128 * u, s[u]);
      } else if constexpr (BIAS == 2) {
        const int codes = lds_at(sm) + st * STAGE + 2 * TILE + 4 * P.seg, first = lds_read<int>(codes);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 c = lds_read<i32x4>(codes + 64 * half + 128 * u + 16 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][4 * g + e] = lds_read<float>(seg + 4 * (c[e] - first));
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
      }
    }
    {
      const int rb = opaque(fr);
#pragma unroll
      for (int k = 0; k < NM; ++k) f[k] = rd.row(rb, k, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    {
      const int rb = opaque(fr);
      phase(f, [&](int k, const frag& a) { s[0] = mma(a, q[k], s[0]); }, [&](int k) { return rd.row(rb, k, HALF); });
    }
    {
      const int cb = opaque(fc);
      phase(f, [&](int k, const frag& a) { s[1] = mma(a, q[k], s[1]); }, [&](int k) { return rd.col(cb, k % NT, k / NT, TILE); });
    }
    if (w64 != ~0ULL) {
      seldom();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned mine = (unsigned)(w64 >> (32 * u)) >> (16 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = (mine >> r) & 1 ? s[u][r] : -INFINITY;
      }
    }
    softmax_step(s, o, m, l, P.c);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      frag p[kPieces<T>][NCS];
      prob_frags<T, NCS>(s[u], p);
      const auto use = [&](int k, const frag& a) {
#pragma unroll
        for (int i = 0; i < kPieces<T>; ++i) o[k % NT] = mma(a, p[i][k / NT], o[k % NT]);
      };
      if (u == 0) {
        const int cb = opaque(fc);
        phase(f, use, [&](int k) { return rd.col(cb, k % NT, k / NT, TILE + HALF); });
      } else {
        last_phase(f, use);
      }
    }
    }
    if (P.stages == 1) {
      __syncthreads();
      if (t + 1 < t1) fetch(t + 1, 0);
    }
    drain();
    __syncthreads();
  }
  l = half_sum(l);
  if (rowv) write_row<T, NT>(P, o, m, l, b, hk, head, qi, part, half);
}

// Few rows: all (at most 32) rows of the query heads that share a key head, row = head in group * Lq + i, so that a single token's heads
// fill one tile.  Bound by reading keys and values.  Each of the four waves walks 32 of the 128 keys of a tile by itself, with its own
// ring of `DEPTH` pieces of keys and of values in LDS: a piece is asked for again as soon as its fragments are in registers, no wave
// waits for another, and 64 KB per block stay in flight or in use (two blocks a CU).  The four running softmaxes are merged through LDS
// at the end.  8 rows of 32765 keys (a tenth hidden), 16 heads on 4, 128 channels, bf16, 483 MB: 97 us, 4.95 TB/s, the rate of a large
// copy (118 us with block-wide tiles of 64 KB, two stages and barriers).  fp32, all keys visible, 1.07 GB: 246 us, 4.4 TB/s (132 KB of LDS at 128
// channels, so one block a CU, and rings of one piece).
//
// BIAS: 0 none, 1 a sequence's, at most kFewBias rows: 32 floats per row come with the keys, 2 any other: read into registers, where
// hipcc's wait for them covers the fills in flight too.
constexpr int kFewBias = 8;
template <typename T, int DP>
struct Few {
  static constexpr int kPiece = 32 * Tile<T, DP>::kRowBytes;
  static constexpr int kDepth = kPiece >= 8192 ? 1 : 8192 / kPiece;
  static constexpr int slot(int bias) { return 2 * kPiece + (bias == 1 ? kFewBias * 128 : 0); }
};
template <typename T, int DP, int BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 || DP <= 64 ? 2 : 1)) void mha_few_k(const FwdP P) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::frag frag;
  typedef Filler<T, DP, 32, 1> Fill;
  constexpr int E = Elem<T>::E, KM = 2 * E, NM = DP / KM, NT = DP / 32, NCS = 32 / KM;
  constexpr int PIECE = Few<T, DP>::kPiece, DEPTH = Few<T, DP>::kDepth, SLOT = Few<T, DP>::slot(BIAS), TK = 128;
  constexpr int NV = Fill::N, NK = NV + (BIAS == 1 ? kFewBias / 2 : 0);               // requests of a piece of values, of keys and bias
  extern __shared__ __attribute__((aligned(512))) char sm[];         // [wave][DEPTH][K | V | bias]; at the end [4][32] m | [4][32] l | [32][DP + 1] o
  const so_mha_desc& D = P.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int G = D.Hq / D.Hk, rows = G * D.Lq;
  const BlockOf blk = block_of(D.B, D.Hk, P.parts);
  const int b = blk.b, hk = blk.hk, part = blk.idx;
  const bool rowv = li < rows;
  const int head = hk * G + (rowv ? li / D.Lq : 0), qi = rowv ? li % D.Lq : 0;

  const unsigned long long* words = D.words ? (const unsigned long long*)D.words + (size_t)b * D.nwords : nullptr;
  int wlo, whi;
  word_range(words, D.Lk, lane, wlo, whi);
  int t0 = wlo / 2, t1 = (whi + 1) / 2;
  if (P.parts > 1) {
    const int lo = t0, n = t1 > t0 ? t1 - t0 : 0;
    t0 = lo + (int)((long long)n * part / P.parts);
    t1 = lo + (int)((long long)n * (part + 1) / P.parts);
  }

  frag q[NM];
  {
    const T* qr = (const T*)D.q + (size_t)b * D.sqb + (size_t)qi * D.sql + (size_t)head * D.sqh;
#pragma unroll
    for (int m = 0; m < NM; ++m) q[m] = as_frag<T>(load_chunk<T>(qr, 2 * m + half, rowv && (2 * m + half) * E < D.D));
  }
  const T* kb = (const T*)D.k + (size_t)b * D.skb + (size_t)hk * D.skh;
  const T* vb = (const T*)D.v + (size_t)b * D.svb + (size_t)hk * D.svh;
  const Fill fk(D.D, (unsigned)(D.skl * sizeof(T)), lane), fv(D.D, (unsigned)(D.svl * sizeof(T)), lane);
  const int mine = wave * DEPTH * SLOT;
  const Reader<T, DP> rd(sm + mine, lane);
  KeyWords kw(words, D.nwords, D.Lk, lane);
  const auto bits_of = [&](int t) { return (unsigned)(kw.get(2 * t + (wave >> 1)) >> (32 * (wave & 1))); };
  const float* bias = nullptr;      // of the lane's row
  if constexpr (BIAS == 2) bias = D.bias + (size_t)head * D.V + D.code_max - D.code[D.q_start + qi];
  i32x4 brs = {};
  unsigned boff[kFewBias / 2];      // rows 2 j and 2 j + 1 of the block, one key per lane
  if constexpr (BIAS == 1) {
#pragma unroll
    for (int j = 0; j < kFewBias / 2; ++j) {
      const int r = 2 * j + half;
      boff[j] = r < rows ? 4u * (unsigned)((hk * G + r / D.Lq) * (long long)D.V + D.code_max - (D.q_start + r % D.Lq) + li) : 0x80000000u;
    }
    brs = rsrc_of(D.bias, (unsigned)(4LL * D.Hq * D.V));
  }
  const auto fetch_k = [&](int t, int at, unsigned bits) {
    const size_t key0 = (size_t)t * TK + 32 * wave;
    if constexpr (BIAS == 1) {
#pragma unroll
      for (int j = 0; j < kFewBias / 2; ++j) dma4(brs, lds_at(sm) + at + 2 * PIECE + 256 * j, boff[j] + 4u * (unsigned)key0);
    }
    fk.fill(sm + at, kb + key0 * D.skl, bits | 0xFFFFFFFF00000000ULL, 0, 0);
  };
  const auto fetch_v = [&](int t, int at, unsigned bits) {
    fv.fill(sm + at + PIECE, vb + ((size_t)t * TK + 32 * wave) * D.svl, bits | 0xFFFFFFFF00000000ULL, 0, 0);
  };

  frag f[NM];
  f32x16 o[NT], s[1];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < NM; ++k) settle(q[k]);
  unsigned ring[DEPTH];             // visible keys of the pieces in the ring
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) {
    ring[i] = 0;
    if (t0 + i < t1) {
      ring[i] = bits_of(t0 + i);
      fetch_k(t0 + i, mine + i * SLOT, ring[i]);
      fetch_v(t0 + i, mine + i * SLOT, ring[i]);
    }
  }
  int slot = 0;
  for (int t = t0; t < t1; ++t) {
    const bool more = t + DEPTH < t1;
    const unsigned w = ring[0];
#pragma unroll
    for (int i = 0; i + 1 < DEPTH; ++i) ring[i] = ring[i + 1];
    if constexpr (BIAS == 2) {
      const int key0 = t * TK + 32 * wave + 16 * half;
      if (D.linear) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4u v = *reinterpret_cast<const f32x4u*>(bias + key0 + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][4 * g + e] = v[e];
        }
      } else {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 v = *reinterpret_cast<const i32x4*>(D.code + key0 + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][4 * g + e] = bias[v[e]];
        }
      }
    }
    // requests younger than this piece's keys: its values and the pieces behind it (near the end the ring is not full: wait for all)
    if (more) arrived<NV + (DEPTH - 1) * (NK + NV)>();
    else arrived<0>();
    {
      const int rb = opaque(rd.rows + slot * SLOT);
#pragma unroll
      for (int k = 0; k < NM; ++k) f[k] = rd.row(rb, k, 0);
    }
    if constexpr (BIAS == 1) {      // lanes behind the last row read a row of the ring that nobody uses
      const int at = lds_at(sm) + mine + slot * SLOT + 2 * PIECE + 128 * (li & (kFewBias - 1)) + 64 * half;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = lds_read<f32x4>(at + 16 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][4 * g + e] = v[e];
      }
    } else if constexpr (BIAS == 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
    }
    if (more) {
      ring[DEPTH - 1] = bits_of(t + DEPTH);
      lds_done();
      fetch_k(t + DEPTH, mine + slot * SLOT, ring[DEPTH - 1]);
    }
#pragma unroll
    for (int k = 0; k < NM; ++k) s[0] = mma(f[k], q[k], s[0]);
    if (w != ~0u) {
      seldom();
      const unsigned seen = w >> (16 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = (seen >> r) & 1 ? s[0][r] : -INFINITY;
    }
    softmax_step(s, o, m, l, P.c);
    frag p[kPieces<T>][NCS];
    prob_frags<T, NCS>(s[0], p);
    if (more) arrived<DEPTH * NK + (DEPTH - 1) * NV>();
    else arrived<0>();
    {
      const int cb = opaque(rd.cols + slot * SLOT);
#pragma unroll
      for (int k = 0; k < NM; ++k) f[k] = rd.col(cb, k % NT, k / NT, PIECE);
    }
    if (more) {
      lds_done();
      fetch_v(t + DEPTH, mine + slot * SLOT, ring[DEPTH - 1]);
    }
    last_phase(f, [&](int k, const frag& a) {
#pragma unroll
      for (int i = 0; i < kPieces<T>; ++i) o[k % NT] = mma(a, p[i][k / NT], o[k % NT]);
    });
    slot = slot + 1 < DEPTH ? slot + 1 : 0;
  }
  l = half_sum(l);
  __syncthreads();

  // merge the four waves' softmaxes: statistics first, then each wave adds its scaled rows in turn
  float* stats = reinterpret_cast<float*>(sm);
  if (half == 0) {
    stats[32 * wave + li] = m;
    stats[128 + 32 * wave + li] = l;
  }
  __syncthreads();
  float mn = -INFINITY, ln = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) mn = fmaxf(mn, stats[32 * w + li]);
  const float ms = mn == -INFINITY ? 0.f : mn;
#pragma unroll
  for (int w = 0; w < 4; ++w) ln += stats[128 + 32 * w + li] * exp2_(stats[32 * w + li] - ms);
  const float scale = exp2_(m - ms);
  float* os = stats + 256;
  for (int w = 0; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int v = 0; v < NT; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float* at = os + li * (DP + 1) + 32 * v + acc_row(r, half);
          const float x = o[v][r] * scale;
          *at = w == 0 ? x : *at + x;
        }
    }
    __syncthreads();
  }
  if (wave != 0 || !rowv) return;
#pragma unroll
  for (int v = 0; v < NT; ++v)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[v][r] = os[li * (DP + 1) + 32 * v + acc_row(r, half)];
  write_row<T, NT>(P, o, mn, ln, b, hk, head, qi, part, half);
}

// Joining the parts of a row: o = sum_p w_p o_p / sum_p w_p l_p with w_p = 2^(m_p - max m), in a fixed order.  Bound by the latency of
// one round of reads, so everything is requested before the first use.
// 128 rows of 16 parts 4.9 us (13 as a wave per row that reads its weights first), 32784 rows of 64 channels in 3 parts 10 us (19).
// four channels of a joined row
template <typename T>
__device__ __forceinline__ void write_joined(const so_mha_desc& D, long long at, int c, f32x4 x, float mn, float l) {
  const int rows = D.Hq / D.Hk * D.Lq, bh = (int)(at / rows), row = (int)(at - (long long)bh * rows), b = bh / D.Hk, hk = bh - b * D.Hk;
  const int head = hk * (D.Hq / D.Hk) + row / D.Lq, qi = row % D.Lq;
  const size_t orow = (((size_t)b * D.Lq + qi) * D.Hq + head) * D.D;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] *= inv;
    y[e] = (T)x[e];
  }
  *reinterpret_cast<t4*>((T*)D.o + orow + c) = y;
  if (D.o_f32) *reinterpret_cast<f32x4*>(D.o_f32 + orow + c) = x;
  if (D.stats && c == 0) write_stats(D, b, head, qi, mn, l, inv);
}

// up to kJoin parts: half a wave per row, four channels per lane
constexpr int kJoin = 8;
template <typename T>
__global__ __launch_bounds__(256) void mha_join_k(const FwdP P) {
  const so_mha_desc& D = P.d;
  const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), n = (long long)D.B * D.Hq * D.Lq;
  const int c = 4 * (threadIdx.x & 31);
  if (at >= n || c >= D.D) return;
  const float* ml = D.part_ml + 2 * at * P.parts;
  const float* po = D.part_o + at * P.parts * D.D + c;
  float m[kJoin], l[kJoin], mn = -INFINITY, ln = 0.f;
  f32x4 o[kJoin], x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < kJoin; ++p) {
    const int i = p < P.parts ? p : 0;
    m[p] = p < P.parts ? ml[2 * i] : -INFINITY;
    l[p] = p < P.parts ? ml[2 * i + 1] : 0.f;
    o[p] = p < P.parts ? *reinterpret_cast<const f32x4*>(po + (size_t)i * D.D) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int p = 0; p < kJoin; ++p) mn = fmaxf(mn, m[p]);
  const float ms = mn == -INFINITY ? 0.f : mn;
#pragma unroll
  for (int p = 0; p < kJoin; ++p) {
    const float w = exp2_(m[p] - ms);
    ln += l[p] * w;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += o[p][e] * w;
  }
  write_joined<T>(D, at, c, x, mn, ln);
}

// more parts (at most 256; few rows): a block per row, eight parts at a time
template <typename T>
__global__ __launch_bounds__(256) void mha_join_many_k(const FwdP P) {
  __shared__ float weight[256], sums[2];
  __shared__ f32x4 piece[8][32];
  const so_mha_desc& D = P.d;
  const long long at = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, g = tid >> 5, c = 4 * (tid & 31);
  const float* ml = D.part_ml + 2 * at * P.parts;
  const float* po = D.part_o + at * P.parts * D.D + c;
  f32x4 o[4], x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = g + 8 * j;
    o[j] = p < P.parts && c < D.D ? *reinterpret_cast<const f32x4*>(po + (size_t)p * D.D) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (tid < 64) {      // lane p holds the statistics of parts p, p + 64, ...
    float m[4], l[4], mn = -INFINITY, ln = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = lane + 64 * i;
      m[i] = p < P.parts ? ml[2 * p] : -INFINITY;
      l[i] = p < P.parts ? ml[2 * p + 1] : 0.f;
      mn = fmaxf(mn, m[i]);
    }
    mn = so_wave_max(mn);
    const float ms = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = exp2_(m[i] - ms);
      weight[lane + 64 * i] = w;
      ln += l[i] * w;
    }
    ln = so_wave_sum(ln);
    if (lane == 0) {
      sums[0] = mn;
      sums[1] = ln;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += o[j][e] * weight[g + 8 * j];
  if (c < D.D)
    for (int p = g + 32; p < P.parts; p += 8) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(po + (size_t)p * D.D);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += v[e] * weight[p];
    }
  piece[g][tid & 31] = x;
  __syncthreads();
  if (tid >= 32 || c >= D.D) return;
#pragma unroll
  for (int i = 1; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += piece[i][tid][e];
  write_joined<T>(D, at, c, x, sums[0], sums[1]);
}

// bias[h][v] = table[lut[v]][h] / scale, finite values kept finite; words[b][w] = bits of the mask bytes
struct PrepP {
  const float* table;
  const int* lut;
  const unsigned char* mask;
  float* bias;
  unsigned long long* words;
  long long mask_sb;
  int V, H, B, Lk, nwords, bias_blocks;
  float inv_scale, top;
};
__global__ __launch_bounds__(256) void mha_prep_k(const PrepP p) {
  if ((int)blockIdx.x < p.bias_blocks) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= p.V) return;
    const float* row = p.table + (size_t)p.lut[v] * p.H;
    for (int h = blockIdx.y; h < p.H; h += gridDim.y) {
      float x = row[h];
      if (x > -INFINITY && x < INFINITY) x = fminf(fmaxf(x * p.inv_scale, -p.top), p.top);
      p.bias[(size_t)h * p.V + v] = x;
    }
    return;
  }
  if (blockIdx.y) return;
  const int lane = threadIdx.x & 63;
  const long long i = (long long)(blockIdx.x - p.bias_blocks) * 4 + (threadIdx.x >> 6);
  if (i >= (long long)p.B * p.nwords) return;
  const int b = (int)(i / p.nwords), w = (int)(i - (long long)b * p.nwords), key = 64 * w + lane;
  const unsigned long long bits = __ballot(key < p.Lk && p.mask[b * p.mask_sb + key] != 0);
  if (lane == 0) p.words[i] = bits;
}

template <typename K>
int start(K k, const FwdP& p, size_t lds, long long blocks, hipStream_t st) {
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), lds, st, p);
  return SO_LAUNCH_CHECK();
}
template <typename T, int DP>
int launch(FwdP p, bool few, hipStream_t st) {
  constexpr size_t row = Tile<T, DP>::kRowBytes;
  const long long groups = (long long)p.d.B * p.d.Hk;
  if (few) {
    constexpr size_t merge = (256 + 32 * (DP + 1)) * 4;
    typedef Few<T, DP> F;
    const auto lds = [&](int bias) { const size_t n = 4 * F::kDepth * F::slot(bias); return n > merge ? n : merge; };
    if (!p.d.bias) return start(mha_few_k<T, DP, 0>, p, lds(0), groups * p.parts, st);
    // the expanded bias is addressed with 31 bits
    if (p.d.linear && p.d.Hq / p.d.Hk * p.d.Lq <= kFewBias && 4LL * p.d.Hq * p.d.V < 0x7fffffffLL)
      return start(mha_few_k<T, DP, 1>, p, lds(1), groups * p.parts, st);
    return start(mha_few_k<T, DP, 2>, p, lds(2), groups * p.parts, st);
  }
  const int w = p.d.linear ? 1 : p.d.width;
  p.seg = p.d.bias ? (code_span(128, w) + code_span(64, w) + 1 + 63) / 64 * 64 : 0;
  const size_t stage = (2 * 64 * row + 4 * (size_t)p.seg + (p.d.bias && !p.d.linear ? 256 : 0) + 511) & ~(size_t)511;   // the readers' XOR needs whole 512s
  p.stage_bytes = (int)stage;
  p.stages = 2 * stage <= kLds ? 2 : 1;
  const long long blocks = groups * (p.d.Hq / p.d.Hk) * p.row_tiles * p.parts;
  const size_t lds = p.stages * stage;
  if (!p.d.bias) return start(mha_fwd_k<T, DP, 0>, p, lds, blocks, st);
  return p.d.linear ? start(mha_fwd_k<T, DP, 1>, p, lds, blocks, st) : start(mha_fwd_k<T, DP, 2>, p, lds, blocks, st);
}
template <typename T>
int launch_d(const FwdP& p, bool few, hipStream_t st) {
  if (p.d.D <= 32) return launch<T, 32>(p, few, st);
  if (p.d.D <= 64) return launch<T, 64>(p, few, st);
  if (p.d.D <= 96) return launch<T, 96>(p, few, st);
  return launch<T, 128>(p, few, st);
}

// few rows: everything that shares a key head fits one 32-row tile
bool is_few(const so_mha_desc* d) { return (long long)(d->Hq / d->Hk) * d->Lq <= 32; }

}  // namespace

// shape, type and alignment rules that all entry points share
int so_mha_check(const so_mha_desc* d) {
  if (!d || (d->dtype != SO_F32 && d->dtype != SO_BF16)) return SO_ERR_SHAPE;
  if (d->B < 1 || d->Hq < 1 || d->Hk < 1 || d->Hq % d->Hk || d->Lq < 1 || d->Lk < 1 || d->D < 1 || d->D > 128) return SO_ERR_SHAPE;
  if ((long long)d->B * d->Hk > 0x7fffffffLL || (long long)(d->Hq / d->Hk) * d->Lq > 0x7fffff00LL || d->Lk > 0x7fffff00) return SO_ERR_SHAPE;
  if (!(d->scale > 0.f) || d->nwords != (d->Lk + 63) / 64) return SO_ERR_SHAPE;
  const int E = d->dtype == SO_F32 ? 4 : 8;
  if (d->D % E) return SO_ERR_ALIGN;
  // a tile's rows lie within 2^31 bytes of its first
  if (d->skl < 0 || d->svl < 0 || d->sql < 0 || d->skl * 4 * 128 >= (1LL << 31) || d->svl * 4 * 128 >= (1LL << 31) || d->sql * 4 * 128 >= (1LL << 31) ||
      (long long)d->Hq * d->D * 4 * 128 >= (1LL << 31)) return SO_ERR_SHAPE;
  const long long s[] = {d->sqb, d->sql, d->sqh, d->skb, d->skl, d->skh, d->svb, d->svl, d->svh};
  for (long long x : s)
    if (x % E) return SO_ERR_ALIGN;
  if ((((uintptr_t)d->q) | ((uintptr_t)d->k) | ((uintptr_t)d->v) | ((uintptr_t)d->o) | ((uintptr_t)d->o_f32)) & 15) return SO_ERR_ALIGN;
  if (d->bias && (!d->code || (((uintptr_t)d->code) & 15) || d->V != 2 * d->code_max + 1 || d->q_start < 0)) return SO_ERR_SHAPE;
  if (d->bias && !d->linear && (d->width < 1 || d->width > 512)) return SO_ERR_SHAPE;
  if (d->bias && (d->q_start + (long long)d->Lq > d->tokens || d->Lk > d->tokens)) return SO_ERR_SHAPE;
  return 0;
}

double mha_tiles(int n) { return n / 128 + (n % 128 + 31) / 32 * 0.25; }

int mha_split_parts(double blocks, double block_us, double join_us, double part_bytes, double rate, int most, double gain) {
  // 66 MB of partial sums (two 64 x 36 maps, 7 parts) were joined at 16 TB/s, 134 MB (2 x 4097 tokens, 16 heads of 128, 2 parts) at 3.9
  constexpr double kCached = 100e6, kCopy = 4.9e6;
  int best = 1;
  double least = 0;
  for (int p = 1; p <= 8 && (p == 1 || p <= most); ++p) {
    const double bytes = part_bytes * p, at = bytes / 2 > kCached && rate > kCopy ? kCopy : rate;
    const double t = ceil(blocks * p / 256) / p * block_us + (p > 1 ? join_us + bytes / at : 0.0);
    if (p == 1 || t < gain * least) {
      best = p;
      least = t;
    }
  }
  return best;
}

extern "C" {

int so_mha_desc_bytes(void) { return (int)sizeof(so_mha_desc); }

int so_mha_prep(const float* table, const void* lut, int V, int H, float scale, float* bias, const void* mask, long long mask_sb, int B,
                int Lk, void* words, void* stream) {
  if ((table && (V < 1 || H < 1 || !lut || !bias)) || (mask && (B < 1 || Lk < 1 || !words)) || !(scale > 0.f)) return SO_ERR_SHAPE;
  PrepP p = {};
  p.table = table; p.lut = (const int*)lut; p.mask = (const unsigned char*)mask; p.bias = bias; p.words = (unsigned long long*)words;
  p.mask_sb = mask_sb; p.V = V; p.H = H; p.B = B; p.Lk = Lk; p.nwords = (Lk + 63) / 64;
  p.bias_blocks = table ? (V + 255) / 256 : 0;
  p.inv_scale = 1.f / scale;
  // Finite entries are kept within +-2^30 in the kernels' log2 units: exp2(fma(acc, c, -m)) sees the rounding of m = max(acc c), at most
  // 2^-24 of it, as a common factor of a row - at 2^30 that is 2^64, still far from overflow - which the row's sum carries as well.
  p.top = 1073741824.f / (scale * kLog2e);
  const long long mb = mask ? ((long long)B * p.nwords + 3) / 4 : 0;
  if (p.bias_blocks + mb == 0) return 0;
  if (p.bias_blocks + mb > 0x7fffffffLL) return SO_ERR_SHAPE;
  hipLaunchKernelGGL(mha_prep_k, dim3((unsigned)(p.bias_blocks + mb), table ? (H < 16 ? H : 16) : 1), dim3(256), 0, (hipStream_t)stream, p);
  return SO_LAUNCH_CHECK();
}

// Parts of the key axis.  Few rows (bound by reading keys): enough blocks to give every CU two, at least two tiles to a part.  Many rows:
// blocks that share a CU share its matrix pipes, so the pass takes as long as the CU with most blocks - ceil(blocks parts / 256) / parts
// of a block's time - and joining costs a launch and 8 bytes per element and part; the cheapest of up to eight parts is taken.  (fp32, 2 x
// 2049 tokens, 8 heads of 64, 272 blocks: 292, 247, 220, 226 us with 1, 2, 3, 4 parts; bf16, 4 x 600 tokens, 16 heads of 128, 320 blocks: 45,
// 53, 59, 62 us; one head of 1024: 26, 20, 17, 15 us; 2 x 4097 tokens, 16 heads of 128: 599 and 606 us with 1 and 2 or 3 parts, for 134 MB or
// more of partial sums.)
int so_mha_parts(const void* desc) {
  const so_mha_desc* d = (const so_mha_desc*)desc;
  const int err = so_mha_check(d);
  if (err) return err;
  if (is_few(d)) {
    const long long blocks = (long long)d->B * d->Hk;
    const int tiles = (d->Lk + 127) / 128;
    long long parts = (512 + blocks - 1) / blocks;
    if (parts > tiles / 2) parts = tiles / 2;
    return parts < 2 ? 1 : (int)(parts > 256 ? 256 : parts);
  }
  // a map's bias is looked up value by value, bf16 probabilities are three products for one: 2 x 2304 tokens of a 64 x 36 map, 8 heads of 64,
  // 288 blocks, training: 116 us whole, 83 + 10 in two parts, 69 + 12 in seven (the join reads from caches)
  const double rate = (d->dtype == SO_BF16 ? 0.75 : 1.0) * (d->bias && !d->linear ? 0.6 : 1.0), rows = (double)d->B * d->Hq * d->Lq;
  return mha_split_parts((double)d->B * d->Hq * mha_tiles(d->Lq), mha_us(4.0 * 128 * d->D * d->Lk, d->dtype) / rate, 8.0,
                         rows * d->D * 8, 12e6, d->Lk / 128, 0.95);
}

int so_mha_fwd(const void* desc, void* stream) {
  const so_mha_desc* d = (const so_mha_desc*)desc;
  const int parts = so_mha_parts(d);
  if (parts < 0) return parts;
  if (!d->q || !d->k || !d->v || !d->o || (parts > 1 && (!d->part_o || !d->part_ml || (((uintptr_t)d->part_o) & 15)))) return SO_ERR_SHAPE;
  FwdP p = {};
  p.d = *d;
  p.parts = parts;
  p.c = d->scale * kLog2e;
  const bool few = is_few(d);
  p.row_tiles = (d->Lq + 127) / 128;
  if ((long long)d->B * d->Hq * p.row_tiles * parts > 0x7fffffffLL) return SO_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  const int err = d->dtype == SO_F32 ? launch_d<float>(p, few, st) : launch_d<__bf16>(p, few, st);
  if (err || parts == 1) return err;
  const long long rows = (long long)d->B * d->Hq * d->Lq, n = parts > kJoin ? rows : (rows + 7) / 8;
  if (n > 0x7fffffffLL) return SO_ERR_SHAPE;
  void (*const join)(FwdP) = parts > kJoin ? (d->dtype == SO_F32 ? mha_join_many_k<float> : mha_join_many_k<__bf16>)
                                           : (d->dtype == SO_F32 ? mha_join_k<float> : mha_join_k<__bf16>);
  hipLaunchKernelGGL(join, dim3((unsigned)n), dim3(256), 0, st, p);
  return SO_LAUNCH_CHECK();
}

}  // extern "C"
