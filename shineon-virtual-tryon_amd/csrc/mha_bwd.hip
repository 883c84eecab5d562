// Multi-head attention with a learned relative position bias, backward, gfx950.
//
//   P = exp2(c s - m) / l,  delta_i = sum_c do_ic o_ic,  dS = P (do v^T - delta),
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T do,  dtable[r][h] = sum of dS_h over the pairs of bucket r
//
// Two passes over the score matrix, each rebuilding P from q, k and the saved row statistics, so that every sum has one owner and a
// fixed order (no atomics on global memory): mha_dq_k owns query rows and walks the keys, mha_dkv_k owns keys and walks the query
// rows of all heads that share them.  7 products instead of the 5 of a single pass whose dq would be added up by atomics.
//
// The bias gradient needs dS summed along the diagonals of equal offset.  In mha_dq_k a wave adds the sums of each 32 x 32 piece into
// rings of its own in LDS, indexed by offset modulo the ring, in a fixed order.  As the walk over the keys moves on, offsets that no later
// key can reach are summed over the block's rings and written to the block's strip; mha_dvec_k and mha_drow_k add strips over blocks and
// offsets over buckets.  (LDS float atomics, one ds_add_f32 per register, were the first form: 300 cycles each, two thirds of the whole
// backward pass.)
#include "mha.h"

using namespace mha;

namespace {

struct BwdP {
  so_mha_desc d;
  float c;            // scale * log2 e
  int ring, strip;    // floats of one LDS ring (a power of two) and of one block's strip
  int stages, stage_bytes, qtiles, ktiles;
  int dq_parts, dkv_parts;        // parts of the keys (mha_dq_k) and of the query rows (mha_dkv_k); their sums: d.part_o, joined by mha_sum_k
  long long dkv_at;               // where those of dk, dv begin
  int seg;            // floats of the bias that a tile of 64 and a block of 128 tokens can meet, in whole 64s
};

constexpr int BK = 64;          // keys (mha_dq_k) or query rows (mha_dkv_k) of a tile

template <int CTRL, bool ZERO>
__device__ __forceinline__ float dpp(float old, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, 0xF, 0xF, ZERO));
}

// Diagonal sums of a 16 x 16 piece per row of 16 lanes, in vector instructions: lane j holds query j, s[r] key r.  The running sums move
// one lane up per key (lane j then holds diagonal r - j); what leaves lane 15 is finished and enters lane 0 of a second register, which
// moves along.  At the end run = diagonal 15 - j, fin = diagonal -1 - j (lane 15: zero).
__device__ __forceinline__ void diagonals16(const f32x16& s, float& run, float& fin) {
  constexpr int kShr1 = 0x111, kRor1 = 0x121;
  run = s[0];
  fin = 0.f;
#pragma unroll
  for (int r = 1; r < 16; ++r) {
    fin = dpp<kShr1, false>(dpp<kRor1, true>(0.f, run), fin);
    run = s[r] + dpp<kShr1, true>(0.f, run);
  }
}

// The 16 keys x 32 queries of one half, tokens of a sequence: the diagonals of the second row's run are those of the first row's fin, and
// the first row's run (pend, kept in the second row's lanes) are those of the second row's fin 32 keys further on, where this half of the
// wave works next.  So every call finishes the 32 diagonals in front of its keys: lane l returns diagonal -1 - l against the half's first
// key and the wave's first query.
__device__ __forceinline__ float diagonals(const f32x16& s, float& pend, int li) {
  float run, fin;
  diagonals16(s, run, fin);
  // rows 0 1 2 3 -> first: 0 0 2 2, second: 1 1 3 3
  const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(run), __float_as_uint(run), false, false);
  const float x = fin + (li < 16 ? __uint_as_float(rows[1]) : pend);
  pend = __uint_as_float(rows[0]);
  return x;
}

// The same for tokens of a map.  A row of 16 lanes holds queries of one map row (see map_query) whose codes count up from cq; the half's
// 16 keys from column x of map row y may reach over map rows, and equal token distances are equal offsets only inside one: a pass per map
// row, the other keys zero.  Sums that are zero are not added: their place may belong to offsets that are being written out.
__device__ __forceinline__ void map_diagonals(const f32x16& s, float* ring, int rmask, int y, int x, int width, int cq, int lj) {
  int from = 0;
  while (__any(from < 16)) {
    const int to = from + width - x < 16 ? from + width - x : 16;
    float run, fin;
    if (__all(from == 0 && to == 16)) {
      diagonals16(s, run, fin);
    } else {
      const int mask = (1 << to) - (1 << from);
      f32x16 z;
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = __int_as_float(__float_as_int(s[r]) & __builtin_amdgcn_sbfe(mask, r, 1));
      diagonals16(z, run, fin);
    }
    const int v = y * (2 * width - 1) + x - from + 15 - cq - lj;
    if (run != 0.f) ring[v & rmask] += run;
    if (fin != 0.f) ring[(v - 16) & rmask] += fin;
    from = to;
    x = 0;
    ++y;
  }
}

// Query rows of mha_dq_k in a map: map rows are padded to a multiple of 16 lanes.  The i-th of these places, counted from the map row of
// the first query, is column x of map row y.
struct MapQuery { int y, x; };
__device__ __forceinline__ MapQuery map_query(const so_mha_desc& D, int i) {
  const int pitch = (D.width + 15) & ~15, y = i / pitch;
  return MapQuery{D.q_start / D.width + y, i - y * pitch};
}
// codes of the first and the last query that block t of mha_dq_k can hold
__device__ __forceinline__ void block_codes(const so_mha_desc& D, int t, bool map, int& first, int& last) {
  const int q0 = 128 * t, ql = (q0 + 128 < D.Lq ? q0 + 128 : D.Lq) - 1;
  first = D.q_start + q0;
  last = D.q_start + ql;
  if (!map) return;
  const int w = D.width, wc = 2 * w - 1, end = D.q_start + D.Lq - 1;
  const MapQuery a = map_query(D, q0), b = map_query(D, q0 + 127);
  const int lo = D.q_start / w * wc + D.q_start % w, hi = end / w * wc + end % w;
  first = a.y * wc + (a.x < w ? a.x : w - 1);
  last = b.y * wc + (b.x < w ? b.x : w - 1);
  if (first < lo) first = lo;
  if (last > hi) last = hi;
  if (first > last) first = last;
}

// one row of a part's sums
template <int NT>
__device__ __forceinline__ void write_part(float* out, const f32x16 (&x)[NT], int D, float scale, int half) {
#pragma unroll
  for (int v = 0; v < NT; ++v)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * v + 8 * g + 4 * half;
      if (c < D) *reinterpret_cast<f32x4*>(out + c) = f32x4{x[v][4 * g] * scale, x[v][4 * g + 1] * scale, x[v][4 * g + 2] * scale, x[v][4 * g + 3] * scale};
    }
}

// out[i] = sum over parts, in their order; four elements per thread (rows are whole 16-byte chunks)
template <typename T>
__global__ __launch_bounds__(256) void mha_sum_k(const float* part, T* out, long long n, int parts) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 x = *reinterpret_cast<const f32x4*>(part + i);
  for (int p = 1; p < parts; ++p) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(part + p * n + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += y[e];
  }
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (T)x[e];
  *reinterpret_cast<t4*>(out + i) = o;
}

// BIAS: 0 none, 1 tokens of a sequence (offset = key - query), 2 tokens of a map.  Everything a tile needs travels by LDS-DMA: K, V,
// the piece of the expanded bias that its offsets lie in and (maps) the keys' codes; nothing in the loop waits for global memory
// except the one drain per tile.  2 x 4097 tokens, 16 heads on 4 of 128 channels, bf16, with the bias gradient: 557 us, 740 TFLOP/s, matrix and
// vector instructions 41 % of the SIMD cycles each, hardly beside each other; fp32, 4 x 2048, 8 heads of 64: 435 us, 118 TFLOP/s (matrix
// pipes 80 % busy); two 64 x 36 maps, 8 heads of 64, bf16: 154-160 us, 205-212 TFLOP/s, bound by the vector instructions of the bias lookup
// and of map_diagonals (at least 44 % of the cycles; matrix 13 %).
template <typename T, int DP, int BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? (DP <= 64 ? 3 : 2) : DP <= 64 ? 2 : 1)) void mha_dq_k(const BwdP P) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::frag frag;
  constexpr int E = Elem<T>::E, KM = 2 * E, NM = DP / KM, NT = DP / 32, NCS = 32 / KM;
  constexpr int TILE = BK * TL::kRowBytes;
  extern __shared__ __attribute__((aligned(512))) char sm[];          // [stages][K tile | V tile | bias | codes] | rings
  const so_mha_desc& D = P.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, half = lane >> 5;
  const int G = D.Hq / D.Hk;
  const BlockOf blk = block_of(D.B, D.Hk, G * P.qtiles * P.dq_parts);
  const int b = blk.b, hk = blk.hk, part = blk.idx / (G * P.qtiles), gt = blk.idx - part * G * P.qtiles;
  const int head = hk * G + gt / P.qtiles, qtile = gt % P.qtiles, bh = b * D.Hq + head;
  const int q0 = qtile * 128;
  // this lane's query and its code; lanes without one compute with a place in the block's range and zero operands
  int cqf, cql, row = q0 + 32 * wave + li, cq = 0, cq16 = 0;
  block_codes(D, qtile, BIAS == 2, cqf, cql);
  bool rowv = row < D.Lq;
  if constexpr (BIAS == 2) {
    const MapQuery m = map_query(D, row);
    row = m.y * D.width + m.x - D.q_start;
    rowv = m.x < D.width && row >= 0 && row < D.Lq;
    cq = m.y * (2 * D.width - 1) + m.x;
    cq16 = cq - (li & 15);
    cq = cq < cqf ? cqf : cq > cql ? cql : cq;
  } else {
    cq = rowv ? D.q_start + row : cql;
  }
  const int qi = rowv ? row : 0;
  const bool idle = !__any(rowv);      // this wave only helps to fill tiles

  const unsigned long long* words = D.words ? (const unsigned long long*)D.words + (size_t)b * D.nwords : nullptr;
  int t0, t1;
  word_range(words, D.Lk, lane, t0, t1);
  if (P.dq_parts > 1) {
    const int n = t1 > t0 ? t1 - t0 : 0, per = (n + P.dq_parts - 1) / P.dq_parts;
    t0 += part * per;
    t1 = t0 + per < t1 ? t0 + per : t1;
  }

  frag q[NM], go[NM];
  float delta = 0.f;
  {
    const T* qr = (const T*)D.q + (size_t)b * D.sqb + (size_t)qi * D.sql + (size_t)head * D.sqh;
    const size_t orow = (((size_t)b * D.Lq + qi) * D.Hq + head) * D.D;
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const int ch = 2 * m + half;
      const bool on = rowv && ch * E < D.D;
      q[m] = as_frag<T>(load_chunk<T>(qr, ch, on));
      go[m] = as_frag<T>(load_chunk<T>((const T*)D.dout + orow, ch, on));
      if (D.o_f32) {
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
          const f32x4 ov = load_chunk<float>(D.o_f32 + orow, ch * (E / 4) + h, on);
#pragma unroll
          for (int e = 0; e < 4; ++e) delta += (float)go[m][4 * h + e] * ov[e];
        }
      } else {
        const frag ov = as_frag<T>(load_chunk<T>((const T*)D.o + orow, ch, on));
#pragma unroll
        for (int e = 0; e < E; ++e) delta += (float)go[m][e] * (float)ov[e];
      }
    }
    delta = half_sum(delta);
  }
  const size_t stat = ((size_t)b * D.Hq + head) * D.Lq + qi;
  const float m_ref = rowv ? D.stats[stat] : INFINITY, inv = rowv ? D.stats[(size_t)D.B * D.Hq * D.Lq + stat] : 0.f, delta_inv = delta * inv;
  if (rowv && half == 0 && part == 0) D.delta[stat] = -delta;

  // the first offset of tile t's piece of the bias is code(first key) - code(last query)
  const int STAGE = P.stage_bytes;
  const Reader<T, DP> rd(sm, lane);
  constexpr int HALF = 32 * TL::kRowBytes;      // the second 32 rows of a tile
  const int mine_q = BIAS == 0 ? 0 : cql - cq + (BIAS == 1 ? 16 * half : 0);      // this lane's place in a tile's piece of the bias
  const float* bias = BIAS ? D.bias + (size_t)head * D.V + D.code_max - cql : nullptr;

  // bias gradient: rings cleared, strip filled with zeros up to the first offset that the walk can reach
  constexpr int RINGS = 8;
  const bool want = BIAS && D.strips != nullptr;
  float* rings = reinterpret_cast<float*>(sm + P.stages * STAGE);
  float* mine = rings + (2 * wave + half) * P.ring;
  const int qw = D.q_start + q0 + 32 * wave;                         // first token of the wave's rows
  const int rmask = P.ring - 1;
  const int v0 = -cql;                                                 // code[0] = 0
  float* strip = want ? D.strips + (((size_t)bh * P.qtiles + qtile) * P.dq_parts + part) * P.strip : nullptr;
  int flushed = v0;
  if (want) {
    for (int i = tid; i < RINGS * P.ring; i += 256) rings[i] = 0.f;
    const int first = t0 < t1 ? (BIAS == 1 ? t0 * BK : D.code[t0 * BK]) - cql : v0;
    for (int v = v0 + tid; v < first; v += 256) strip[v - v0] = 0.f;
    flushed = first;
  }
  float pend = 0.f;      // sequences: see diagonals()
  int base = 0;
  auto flush = [&](int upto, int turn) {      // one wave's worth at a time, another wave first every time
    for (int v = flushed + ((tid + 64 * turn) & 255); v < upto; v += 256) {
      float x[RINGS], sum = 0.f;
#pragma unroll
      for (int r = 0; r < RINGS; ++r) x[r] = rings[r * P.ring + (v & rmask)];
#pragma unroll
      for (int r = 0; r < RINGS; ++r) {
        sum += x[r];
        rings[r * P.ring + (v & rmask)] = 0.f;
      }
      strip[v - v0] = sum;
    }
    if (upto > flushed) flushed = upto;
  };

  const T* kb = (const T*)D.k + (size_t)b * D.skb + (size_t)hk * D.skh;
  const T* vb = (const T*)D.v + (size_t)b * D.svb + (size_t)hk * D.svh;
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const Filler<T, DP, BK, 4> fk(D.D, (unsigned)(D.skl * sizeof(T)), tid), fv(D.D, (unsigned)(D.svl * sizeof(T)), tid);
  KeyWords kw(words, D.nwords, D.Lk, lane);
  unsigned long long next = 0;
  auto fetch = [&](int t, int st) {
    next = kw.get(t);
    char* kt = sm + st * STAGE;
    fk.fill(kt, kb + (size_t)t * BK * D.skl, next, 0, wave_u);
    fv.fill(kt + TILE, vb + (size_t)t * BK * D.svl, next, 0, wave_u);
    if constexpr (BIAS == 1) fill_dwords<4>(kt + 2 * TILE, bias + t * BK, BK + cql - cqf, 0x7FFFFFFFu, wave_u, lane);
    if constexpr (BIAS == 2) {
      const int c0 = D.code[t * BK];
      fill_dwords<4>(kt + 2 * TILE, bias + c0, D.code[t * BK + BK - 1] - cqf - (c0 - cql) + 1, 0x7FFFFFFFu, wave_u, lane);
      fill_dwords<4>(kt + 2 * TILE + 4 * P.seg, D.code + t * BK, BK, 0x7FFFFFFFu, (wave_u + 1) & 3, lane);
    }
  };

  frag f[NM];      // NM = NT * NCS: every phase of a piece has as many steps
  f32x16 dq[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[t][r] = 0.f;
  if (t0 < t1) fetch(t0, 0);
#pragma unroll
  for (int m = 0; m < NM; ++m) {
    settle(q[m]);
    settle(go[m]);
  }
  drain();
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int st = P.stages == 2 ? (t - t0) & 1 : 0;
    const int rows = rd.rows + st * STAGE, cols = rd.cols + st * STAGE;
    const int seg = opaque(lds_at(sm) + st * STAGE + 2 * TILE + 4 * mine_q), codes = lds_at(sm) + st * STAGE + 2 * TILE + 4 * P.seg;
    const unsigned long long w64 = next;
    if (P.stages == 2 && t + 1 < t1) fetch(t + 1, st ^ 1);
    // offsets below those of this tile are final, and nothing adds to them any more (a sequence's rings are written up to the last
    // row's first key exclusively)
    if (want && t > t0) flush(BIAS == 1 ? t * BK - D.q_start - q0 - 128 : lds_read<int>(codes) - cql, t & 3);
    if (!idle) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key0 = t * BK + 32 * u;
      f32x16 s, dp;
      if constexpr (BIAS == 1) {
        lds_read16(seg + 128 * u, s);
      } else if constexpr (BIAS == 2) {
        const int first = lds_read<int>(codes);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 c = lds_read<i32x4>(codes + 64 * half + 128 * u + 16 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * g + e] = lds_read<float>(seg + 4 * (c[e] - first));
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = 0.f;
      if (u == 0) {
        const int rb = opaque(rows);
#pragma unroll
        for (int m = 0; m < NM; ++m) f[m] = rd.row(rb, m, TILE);
        __builtin_amdgcn_sched_barrier(0);
      }
      {
        const int rb = opaque(rows);
        phase(f, [&](int m, const frag& a) { dp = mma(a, go[m], dp); }, [&](int m) { return rd.row(rb, m, HALF * u); });
      }
      {
        const int cb = opaque(cols);
        phase(f, [&](int m, const frag& a) { s = mma(a, q[m], s); }, [&](int m) { return rd.col(cb, m % NT, m / NT, HALF * u); });
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_(__builtin_fmaf(s[r], P.c, -m_ref)) * __builtin_fmaf(dp[r], inv, -delta_inv);      // dS
      const unsigned w = (unsigned)(w64 >> (32 * u));
      if (w != ~0u) {
        seldom();
        const unsigned my = w >> (16 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (my >> r) & 1 ? s[r] : 0.f;
      }
      if constexpr (BIAS == 1) {
        if (want) {
          base = key0 + 16 * half - qw;
          mine[(base - 1 - li) & rmask] = diagonals(s, pend, li);
        }
      }
      if constexpr (BIAS == 2) {
        if (want) {
          const int ya = key0 / D.width, xa = key0 - ya * D.width, yb = (key0 + 16) / D.width, xb = key0 + 16 - yb * D.width;
          map_diagonals(s, mine, rmask, half ? yb : ya, half ? xb : xa, D.width, cq16, li & 15);
        }
      }
      frag g[NCS];
#pragma unroll
      for (int c = 0; c < NCS; ++c) to_frag(s, c, g[c]);
      const auto use = [&](int m, const frag& a) { dq[m % NT] = mma(a, g[m / NT], dq[m % NT]); };
      if (u == 0) {
        const int rb = opaque(rows);
        phase(f, use, [&](int m) { return rd.row(rb, m, TILE + HALF); });
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
  if (want) {
    if (t0 < t1) {
      if constexpr (BIAS == 1) {
        if (li >= 16 && !idle) mine[(base + 31 - li) & rmask] = pend;
        __syncthreads();
      }
      const int kl = (t1 * BK < D.Lk ? t1 * BK : D.Lk) - 1;
      flush((BIAS == 1 ? kl : D.code[kl]) - cqf + 1, 0);
    }
    for (int v = flushed + tid; v < v0 + P.strip; v += 256) strip[v - v0] = 0.f;
  }
  if (!rowv) return;
  const size_t orow = ((size_t)b * D.Lq + qi) * D.Hq + head;
  if (P.dq_parts > 1) {
    float* out = D.part_o + ((size_t)part * D.B * D.Lq * D.Hq + orow) * D.D;
    write_part<NT>(out, dq, D.D, D.scale, half);
    return;
  }
  T* out = (T*)D.dq + orow * D.D;
#pragma unroll
  for (int v = 0; v < NT; ++v)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * v + 8 * g + 4 * half;
      if (c < D.D) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (T)(dq[v][4 * g + e] * D.scale);
        *reinterpret_cast<t4*>(out + c) = x;
      }
    }
}

// Owns 128 keys, 32 per wave, and walks the 64-row tiles of the query heads that share them.  Scores are computed with keys in the lanes, so
// P and dS are already operands of dv = P^T do and dk = dS^T q.  fp32 is bound by the matrix pipes (4 x 2048, 8 heads of 64: 602 us, 114 TFLOP/s,
// 78 % busy); bf16 above 64 channels by what one wave per SIMD leaves open (2 x 4097 tokens, 16 heads on 4 of 128: 933 us, 590 TFLOP/s, matrix
// instructions 31 %, vector instructions 23 % of the SIMD cycles).
template <typename T, int DP, int BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && DP <= 64 ? 2 : 1)) void mha_dkv_k(const BwdP P) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::frag frag;
  constexpr int E = Elem<T>::E, KM = 2 * E, NM = DP / KM, NT = DP / 32, NCS = 32 / KM;
  constexpr int TILE = BK * TL::kRowBytes;
  extern __shared__ __attribute__((aligned(512))) char sm[];          // [stages][Q tile | dO tile | m | 1 / l | -delta | bias | codes]
  const so_mha_desc& D = P.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, half = lane >> 5;
  const int G = D.Hq / D.Hk;
  const int STAGE = P.stage_bytes;
  const Reader<T, DP> rd(sm, lane);
  constexpr int HALF = 32 * TL::kRowBytes;
  // samples and heads in turn: the blocks behind a short sample's last key have nothing to do and are spread over all XCDs
  const unsigned groups = D.B * D.Hk;
  const int bh = (int)(blockIdx.x % groups), kp = (int)(blockIdx.x / groups), part = kp / P.ktiles, kt = kp - part * P.ktiles;
  const int b = bh / D.Hk, hk = bh - b * D.Hk;
  const int key = kt * 128 + 32 * wave + li;
  const unsigned long long* words = D.words ? (const unsigned long long*)D.words + (size_t)b * D.nwords : nullptr;
  const int w0 = 2 * kt;
  const unsigned long long wa = tail_word(w0, D.Lk) & (words ? words[w0] : ~0ULL);
  const unsigned long long wb = w0 + 1 < D.nwords ? tail_word(w0 + 1, D.Lk) & (words ? words[w0 + 1] : ~0ULL) : 0ULL;
  const bool keyv = key < D.Lk, vis = ((wave < 2 ? wa : wb) >> (key & 63)) & 1;

  const bool idle = !__any(vis);       // this wave only helps to fill tiles

  frag k[NM], v[NM];
  {
    const T* kr = (const T*)D.k + (size_t)b * D.skb + (size_t)(keyv ? key : 0) * D.skl + (size_t)hk * D.skh;
    const T* vr = (const T*)D.v + (size_t)b * D.svb + (size_t)(keyv ? key : 0) * D.svl + (size_t)hk * D.svh;
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const int ch = 2 * m + half;
      k[m] = as_frag<T>(load_chunk<T>(kr, ch, vis && ch * E < D.D));
      v[m] = as_frag<T>(load_chunk<T>(vr, ch, vis && ch * E < D.D));
    }
  }
  // first key's and last key's codes; the first offset of a tile's piece of the bias is code(first key) - code(last row of the tile)
  const int ckf = BIAS == 2 ? D.code[kt * 128] : kt * 128, ckl = BIAS == 2 ? D.code[kt * 128 + 127] : kt * 128 + 127;
  const int mine_k = BIAS == 2 ? D.code[key] - ckf : 32 * wave + li - 16 * half;

  const int qt = (D.Lq + BK - 1) / BK, all = (wa | wb) ? G * qt : 0;    // a block without a visible key writes zeros
  const int each = (all + P.dkv_parts - 1) / P.dkv_parts;
  const int from = part * each < all ? part * each : all, n = from + each < all ? from + each : all;
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const Filler<T, DP, BK, 4> fq(D.D, (unsigned)(D.sql * sizeof(T)), tid), fg(D.D, (unsigned)((size_t)D.Hq * D.D * sizeof(T)), tid);
  auto fetch = [&](int t, int st) {
    const int head = hk * G + t / qt, q0 = (t % qt) * BK;
    const unsigned long long rows = tail_word(t % qt, D.Lq);
    char* qtile = sm + st * STAGE;
    fq.fill(qtile, (const T*)D.q + (size_t)b * D.sqb + (size_t)head * D.sqh + (size_t)q0 * D.sql, rows, 0, wave_u);
    fg.fill(qtile + TILE, (const T*)D.dout + (((size_t)b * D.Lq + q0) * D.Hq + head) * D.D, rows, 0, wave_u);
    char* stats = qtile + 2 * TILE;      // m | 1 / l | -delta | bias | codes
    const size_t at = ((size_t)b * D.Hq + head) * D.Lq + q0;
    const unsigned left = D.Lq - q0 < BK ? 4 * (D.Lq - q0) : 4 * BK;
    fill_dwords<4>(stats, D.stats + at, BK, left, wave_u, lane);
    fill_dwords<4>(stats + 4 * BK, D.stats + (size_t)D.B * D.Hq * D.Lq + at, BK, left, (wave_u + 1) & 3, lane);
    fill_dwords<4>(stats + 8 * BK, D.delta + at, BK, left, (wave_u + 2) & 3, lane);
    if constexpr (BIAS != 0) {
      const int* cp = D.code + D.q_start + q0;
      const int cl = BIAS == 2 ? cp[BK - 1] : D.q_start + q0 + BK - 1, n = BIAS == 2 ? ckl - cp[0] - (ckf - cl) + 1 : 128 + BK - 1;
      fill_dwords<4>(stats + 12 * BK, D.bias + (size_t)head * D.V + D.code_max + ckf - cl, n, 0x7FFFFFFFu, (wave_u + 3) & 3, lane);
      if constexpr (BIAS == 2) fill_dwords<4>(stats + 12 * BK + 4 * P.seg, cp, BK, 0x7FFFFFFFu, wave_u, lane);
    }
  };

  frag f[NM];
  f32x16 dk[NT], dv[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[t][r] = dv[t][r] = 0.f;
  if (from < n) fetch(from, 0);
#pragma unroll
  for (int m = 0; m < NM; ++m) {
    settle(k[m]);
    settle(v[m]);
  }
  drain();
  __syncthreads();
  for (int t = from; t < n; ++t) {
    const int st = P.stages == 2 ? (t - from) & 1 : 0;
    const int rows = rd.rows + st * STAGE, cols = rd.cols + st * STAGE;
    const int at = lds_at(sm) + st * STAGE + 2 * TILE, stats = opaque(at + 64 * half), seg = opaque(at + 12 * BK + 4 * mine_k);
    if (P.stages == 2 && t + 1 < n) fetch(t + 1, st ^ 1);
    const int q0 = (t % qt) * BK;
    if (!idle) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s, dp;
      if constexpr (BIAS == 1) {      // rows upwards are offsets downwards
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = lds_read<float>(seg + 4 * (BK - 1 - 32 * u - r));
      } else if constexpr (BIAS == 2) {
        const int codes = lds_at(sm) + st * STAGE + 2 * TILE + 12 * BK + 4 * P.seg, last = seg + 4 * lds_read<int>(codes + 4 * (BK - 1));
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 c = lds_read<i32x4>(codes + 64 * half + 128 * u + 16 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * g + e] = lds_read<float>(last - 4 * c[e]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 de = lds_read<f32x4>(stats + 8 * BK + 128 * u + 16 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * g + e] = de[e];
      }
      if (u == 0) {
        const int rb = opaque(rows);
#pragma unroll
        for (int m = 0; m < NM; ++m) f[m] = rd.row(rb, m, TILE);
        __builtin_amdgcn_sched_barrier(0);
      }
      {
        const int rb = opaque(rows);
        phase(f, [&](int m, const frag& a) { dp = mma(a, v[m], dp); }, [&](int m) { return rd.row(rb, m, HALF * u); });
      }
      {
        const int cb = opaque(cols);
        phase(f, [&](int m, const frag& a) { s = mma(a, k[m], s); }, [&](int m) { return rd.col(cb, m % NT, m / NT, TILE + HALF * u); });
      }
      const int rows_left = D.Lq - q0 - 32 * u;
      if (rows_left < 32) {      // rows behind the last query: their bias is whatever lies in front of the expanded table
        seldom();
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 16 * half + r < rows_left ? s[r] : -INFINITY;
      }
      // a hidden key's lane computes like the others (its k and v are zero) and stores zeros at the end
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ms = lds_read<f32x4>(stats + 128 * u + 16 * g), inv = lds_read<f32x4>(stats + 4 * BK + 128 * u + 16 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          s[r] = exp2_(__builtin_fmaf(s[r], P.c, -ms[e])) * inv[e];
          dp[r] *= s[r];
        }
      }
      frag g[NCS];
#pragma unroll
      for (int c = 0; c < NCS; ++c) to_frag(s, c, g[c]);
      {
        const int cb = opaque(cols);
        phase(f, [&](int m, const frag& a) { dv[m % NT] = mma(a, g[m / NT], dv[m % NT]); },
              [&](int m) { return rd.col(cb, m % NT, m / NT, HALF * u); });
      }
#pragma unroll
      for (int c = 0; c < NCS; ++c) to_frag(dp, c, g[c]);
      const auto use = [&](int m, const frag& a) { dk[m % NT] = mma(a, g[m / NT], dk[m % NT]); };
      if (u == 0) {
        const int rb = opaque(rows);
        phase(f, use, [&](int m) { return rd.row(rb, m, TILE + HALF); });
      } else {
        last_phase(f, use);
      }
    }
    }
    if (P.stages == 1) {
      __syncthreads();
      if (t + 1 < n) fetch(t + 1, 0);
    }
    drain();
    __syncthreads();
  }
  if (!keyv) return;
  const size_t at = (((size_t)b * D.Lk + key) * D.Hk + hk) * D.D;
  if (P.dkv_parts > 1) {
    const size_t all_rows = (size_t)D.B * D.Lk * D.Hk * D.D;
    float* pk = D.part_o + P.dkv_at + (size_t)part * all_rows + at;
    if (!vis) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[x][r] = dv[x][r] = 0.f;
    }
    write_part<NT>(pk, dk, D.D, D.scale, half);
    write_part<NT>(pk + P.dkv_parts * all_rows, dv, D.D, 1.f, half);
    return;
  }
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * x + 8 * g + 4 * half;
      if (c < D.D) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 a, bb;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = vis ? (T)(dk[x][4 * g + e] * D.scale) : (T)0.f;
          bb[e] = vis ? (T)dv[x][4 * g + e] : (T)0.f;
        }
        *reinterpret_cast<t4*>((T*)D.dk + at + c) = a;
        *reinterpret_cast<t4*>((T*)D.dv + at + c) = bb;
      }
    }
}

// dvec[h][code_max + v] = sum over samples and query blocks of their strips; 64 offsets x 4 runs of blocks, joined in order
__global__ __launch_bounds__(256) void mha_dvec_k(const BwdP P, float* dvec) {
  __shared__ float red[4][64];
  const so_mha_desc& D = P.d;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, i = blockIdx.x * 64 + tx, h = blockIdx.y, v = i - D.code_max;
  float x = 0.f;
  for (int t = ty; t < P.qtiles; t += 4) {
    int first, last;
    block_codes(D, t, !D.linear, first, last);
    const int at = v + last;
    if (i >= D.V || at < 0 || at >= P.strip) continue;
    const float* p = D.strips + ((size_t)h * P.qtiles + t) * P.dq_parts * P.strip + at;
    for (int b = 0; b < D.B; ++b)
#pragma unroll 4
      for (int i = 0; i < P.dq_parts; ++i) x += p[((size_t)b * D.Hq * P.qtiles * P.dq_parts + i) * P.strip];
  }
  red[ty][tx] = x;
  __syncthreads();
  if (ty == 0 && i < D.V) dvec[(size_t)h * D.V + i] = ((red[0][tx] + red[1][tx]) + red[2][tx]) + red[3][tx];
}

// dtable[r][h] = sum of dvec over the offsets of bucket r; one block per entry
__global__ __launch_bounds__(256) void mha_drow_k(const float* dvec, const int* order, const int* start, int rows, int H, int V,
                                                  float* dtable) {
  __shared__ float red[4];
  const int r = blockIdx.x / H, h = blockIdx.x - r * H;
  const float* dv = dvec + (size_t)h * V;
  float x = 0.f;
#pragma unroll 4
  for (int j = start[r] + threadIdx.x; j < start[r + 1]; j += 256) x += dv[order[j]];
  x = so_block_sum256(x, red);
  if (threadIdx.x == 0) dtable[blockIdx.x] = x;
}

constexpr int kLds = 160 * 1024;

int make(const so_mha_desc* d, BwdP& p) {
  const int err = so_mha_check(d);
  if (err) return err;
  p = BwdP{};
  p.d = *d;
  p.c = d->scale * kLog2e;
  p.qtiles = (d->Lq + 127) / 128;
  if (d->bias && !d->linear) {      // map rows padded to 16 lanes (map_query)
    const int pitch = (d->width + 15) & ~15, rows = (d->q_start + d->Lq - 1) / d->width - d->q_start / d->width + 1;
    if ((long long)rows * pitch > 0x7fffff00LL) return SO_ERR_SHAPE;
    p.qtiles = (rows * pitch + 127) / 128;
  }
  p.ktiles = (d->Lk + 127) / 128;
  const double tiles = d->bias && !d->linear ? p.qtiles : mha_tiles(d->Lq);
  const double rows = (double)d->B * d->Lq * d->Hq * d->D, keys = (double)d->B * d->Lk * d->Hk * d->D;
  // fp32, 2 x 2049 tokens, 8 heads of 64, 272 blocks: mha_dq_k 350 us whole, 221 + 8 us in three parts
  p.dq_parts = mha_split_parts((double)d->B * d->Hq * tiles, mha_us(6.0 * 128 * d->D * d->Lk, d->dtype), 6.0, rows * 8, 4e6, d->Lk / 128, 0.95);
  // (blocks of keys that a mask hides end at once, which the estimate does not know: the rows are only cut for a clear gain.  A training
  // pass whole / cut: bf16, 2 x 4097 tokens, 16 heads on 4, 128 channels 2125 / 1725 us, with a fifth of the keys hidden 1935 / 1530;
  // 9000 tokens, 8 on 4, 64 channels 1127 / 999; fp32, 2 x 2049, 8 of 64 1066 / 870; 1000 tokens, 8 on 1, 128 channels 371 / 164)
  const double q_tiles = (double)d->Lq * (d->Hq / d->Hk) / 128;
  p.dkv_parts = mha_split_parts((double)d->B * d->Hk * mha_tiles(d->Lk), mha_us(8.0 * 128 * 128 * d->D * q_tiles, d->dtype), 6.0, keys * 16, 4e6,
                                q_tiles < 8 ? (int)q_tiles : 8, 0.7);
  p.dkv_at = p.dq_parts > 1 ? (long long)rows * p.dq_parts : 0;
  p.stages = 2;
  if (d->bias) {
    if (d->width < 1) return SO_ERR_SHAPE;
    const int w = d->linear ? 1 : d->width;
    p.seg = (code_span(128, w) + code_span(BK, w) + 1 + 63) / 64 * 64;
    if (p.seg > 2048) return SO_ERR_SHAPE;
  }
  if (d->strips) {
    if (!d->bias) return SO_ERR_SHAPE;
    const int w = d->linear ? 1 : d->width;
    // the offsets that one tile of keys can reach from the block's rows, and those of the tile before still being written out (256
    // cover a sequence: 47 in front of the tile's first key, 128 rows behind it, 64 of the tile before)
    const int need = code_span(128, w) + code_span(BK, w) + code_span(BK + 1, w) + 1;
    p.ring = 256;
    while (p.ring < need) p.ring <<= 1;
    if (p.ring > 2048) return SO_ERR_SHAPE;
    const long long all = (long long)(d->linear ? d->Lk : (d->Lk - 1) / d->width * (2LL * d->width - 1) + d->width) + code_span(128, w) + 1;
    p.strip = (int)all;
  }
  return 0;
}

template <typename K>
int lds_limit(K k, size_t lds) {
  if (lds <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
}

template <typename T>
int sum_parts(const float* part, void* out, long long n, int parts, hipStream_t st) {
  hipLaunchKernelGGL(mha_sum_k<T>, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, part, (T*)out, n, parts);
  return SO_LAUNCH_CHECK();
}

template <typename T, int DP, int BIAS>
int launch(BwdP p, hipStream_t st) {
  typedef Tile<T, DP> TL;
  constexpr size_t tile = (size_t)BK * TL::kRowBytes;
  const size_t piece = BIAS ? 4 * (size_t)(p.seg + (BIAS == 2 ? BK : 0)) : 0;
  const size_t rings = p.d.strips ? (size_t)8 * p.ring * 4 : 0;
  size_t stage = (2 * tile + piece + 511) & ~(size_t)511;      // the readers' XOR needs whole 512s
  p.stages = 2 * stage + rings <= kLds ? 2 : 1;
  size_t lds = p.stages * stage + rings;
  if (lds > kLds) return SO_ERR_SHAPE;
  p.stage_bytes = (int)stage;
  int err = lds_limit(mha_dq_k<T, DP, BIAS>, lds);
  if (err) return err;
  hipLaunchKernelGGL((mha_dq_k<T, DP, BIAS>), dim3((unsigned)((long long)p.d.B * p.d.Hq * p.qtiles * p.dq_parts)), dim3(256), lds, st, p);
  err = SO_LAUNCH_CHECK();
  if (err) return err;
  stage = (2 * tile + 3 * BK * 4 + piece + 511) & ~(size_t)511;
  p.stages = 2 * stage <= kLds ? 2 : 1;
  lds = p.stages * stage;
  p.stage_bytes = (int)stage;
  err = lds_limit(mha_dkv_k<T, DP, BIAS>, lds);
  if (err) return err;
  hipLaunchKernelGGL((mha_dkv_k<T, DP, BIAS>), dim3((unsigned)((long long)p.d.B * p.d.Hk * p.ktiles * p.dkv_parts)), dim3(256), lds, st, p);
  err = SO_LAUNCH_CHECK();
  const long long rows = (long long)p.d.B * p.d.Lq * p.d.Hq * p.d.D, keys = (long long)p.d.B * p.d.Lk * p.d.Hk * p.d.D;
  if (!err && p.dq_parts > 1) err = sum_parts<T>(p.d.part_o, p.d.dq, rows, p.dq_parts, st);
  if (!err && p.dkv_parts > 1) err = sum_parts<T>(p.d.part_o + p.dkv_at, p.d.dk, keys, p.dkv_parts, st);
  if (!err && p.dkv_parts > 1) err = sum_parts<T>(p.d.part_o + p.dkv_at + p.dkv_parts * keys, p.d.dv, keys, p.dkv_parts, st);
  return err;
}
template <typename T, int DP>
int launch_b(const BwdP& p, hipStream_t st) {
  return !p.d.bias ? launch<T, DP, 0>(p, st) : p.d.linear ? launch<T, DP, 1>(p, st) : launch<T, DP, 2>(p, st);
}
template <typename T>
int launch_d(const BwdP& p, hipStream_t st) {
  if (p.d.D <= 32) return launch_b<T, 32>(p, st);
  if (p.d.D <= 64) return launch_b<T, 64>(p, st);
  if (p.d.D <= 96) return launch_b<T, 96>(p, st);
  return launch_b<T, 128>(p, st);
}

}  // namespace

extern "C" {

long long so_mha_strip_floats(const void* desc) {
  if (!desc) return SO_ERR_SHAPE;
  so_mha_desc d = *(const so_mha_desc*)desc;
  float one;
  d.strips = &one;       // only asked whether it is wanted
  BwdP p;
  const int err = make(&d, p);
  return err ? err : (long long)d.B * d.Hq * p.qtiles * p.dq_parts * p.strip;
}

long long so_mha_bwd_floats(const void* desc) {
  if (!desc) return SO_ERR_SHAPE;
  const so_mha_desc& d = *(const so_mha_desc*)desc;
  BwdP p;
  const int err = make(&d, p);
  return err ? err : p.dkv_at + (p.dkv_parts > 1 ? 2LL * p.dkv_parts * d.B * d.Lk * d.Hk * d.D : 0);
}

int so_mha_bwd(const void* desc, void* stream) {
  const so_mha_desc* d = (const so_mha_desc*)desc;
  BwdP p;
  const int err = make(d, p);
  if (err) return err;
  if (!d->q || !d->k || !d->v || !d->o || !d->dout || !d->dq || !d->dk || !d->dv || !d->stats || !d->delta) return SO_ERR_SHAPE;
  if ((((uintptr_t)d->dout) | ((uintptr_t)d->dq) | ((uintptr_t)d->dk) | ((uintptr_t)d->dv)) & 15) return SO_ERR_ALIGN;
  if ((p.dq_parts > 1 || p.dkv_parts > 1) && (!d->part_o || (((uintptr_t)d->part_o) & 15))) return SO_ERR_SHAPE;
  const long long dq_blocks = (long long)d->B * d->Hq * p.qtiles * p.dq_parts, dkv_blocks = (long long)d->B * d->Hk * p.ktiles * p.dkv_parts;
  if (dq_blocks > 0x7fffffffLL || dkv_blocks > 0x7fffffffLL) return SO_ERR_SHAPE;
  return d->dtype == SO_F32 ? launch_d<float>(p, (hipStream_t)stream) : launch_d<__bf16>(p, (hipStream_t)stream);
}

int so_mha_dtable(const void* desc, const void* order, const void* start, int rows, float* dvec, float* dtable, void* stream) {
  const so_mha_desc* d = (const so_mha_desc*)desc;
  BwdP p;
  const int err = make(d, p);
  if (err) return err;
  if (!d->strips || !order || !start || rows < 1 || !dvec || !dtable || d->Hq > 65535 || (long long)rows * d->Hq > 0x7fffff00LL)
    return SO_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(mha_dvec_k, dim3((d->V + 63) / 64, d->Hq), dim3(256), 0, st, p, dvec);
  int e = SO_LAUNCH_CHECK();
  if (e) return e;
  hipLaunchKernelGGL(mha_drow_k, dim3(rows * d->Hq), dim3(256), 0, st, dvec, (const int*)order, (const int*)start, rows, d->Hq,
                     d->V, dtable);
  return SO_LAUNCH_CHECK();
}

}  // extern "C"
