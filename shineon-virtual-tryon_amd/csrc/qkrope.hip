// RMS norm of every query and key head and the rotation by the token's position, in one pass, forward and backward, gfx950.
//
//   n = x r w,  r = (mean x^2 + eps)^(-1/2)   over the D channels of one head;   with (a, b) = (n_i, n_{i + R/2}), i < R/2:
//   y_i = a cos_i - b sin_i,   y_{i + R/2} = b cos_i + a sin_i,   channels R .. D - 1 unrotated
// backward: dn = the inverse rotation of dy;  dw = sum over rows dn x r;  g = dn w;  dx = r (g - x r mean(g x r)).
//
// HBM-bound: x is read once and y written once (backward: x and dy read, dx written); r is recomputed in the backward pass from the
// x it needs anyway.  A head row belongs to a group of lanes; a lane holds a vector of the first half of the rotated channels and the
// vector of the second half that turns with it, so the rotation needs no exchange and the sums are a few lane swaps inside the group.
// Channels behind R are dealt out as vector pairs the same way.
#include "common.h"
#include "../../include/shineon_hip.h"

namespace {

struct Side {                      // the queries or the keys
  const void* x;
  const void* dy;                  // backward; dense [B][L][H][D]
  void* y;                         // forward: y, backward: dx; dense
  const float* w;
  float* part;                     // backward: [blocks][D] partial sums of dw
  long long sb, sl, sh;            // strides of x in elements
  int H, blocks;
};

struct QkP {
  Side s[2];
  const float* cosv;
  const float* sinv;               // [P][R / 2]
  const void* pos;                 // token positions, or null: the token's index in its sequence
  long long P, pos_sb, pos_sl, start;
  int pos64, B, L, D, R, lanes;    // lanes of one head row (a power of two)
  float eps;
};

// heads of an item and blocks of a side in the backward pass.  2 x 8191 tokens, 20 heads of 128, bf16: forward 38 us with 4 heads, 56 with
// one (4.5 TB/s); backward 61 us with 2 heads and 512 blocks (4.2 TB/s), 66 with 1024, 70 with one head, 91 with 4 (registers)
constexpr int kHeadsFwd = 4, kHeadsBwd = 2, kBlocksBwd = 512;

template <typename T, int V> struct VecOf { typedef T t __attribute__((ext_vector_type(V))); };
template <typename T> struct VecOf<T, 1> { struct t { T v; __device__ T& operator[](int) { return v; } __device__ T operator[](int) const { return v; } }; };

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// the angle row of a token; -1: a position outside the table (its outputs become NaN, nothing is read out of range)
__device__ __forceinline__ long long angle_row(const QkP& p, int b, int l) {
  long long at = p.start + l;
  if (p.pos) {
    const long long o = b * p.pos_sb + l * p.pos_sl;
    at = p.pos64 ? ((const long long*)p.pos)[o] : (long long)((const int*)p.pos)[o];
  }
  return at >= 0 && at < p.P ? at : -1;
}

// A group of lanes takes U heads of one token at a time: the angles (twice the bytes of a bf16 head) are read once for them, and their
// loads are in flight together.  Items =
// (token, U heads) are stepped by carries; a division per item costs as much as a head.
template <typename T, int V, bool BWD, int U>
__global__ __launch_bounds__(256) void qk_norm_rotary_k(const QkP p) {
  typedef typename VecOf<T, V>::t vec;
  const Side& s = p.s[blockIdx.y];
  if ((int)blockIdx.x >= s.blocks) return;
  const int g = threadIdx.x / p.lanes, slot = threadIdx.x & (p.lanes - 1), per = 256 / p.lanes;
  const int half = p.R / 2, turning = half / V, slots = p.D / (2 * V);
  const bool live = slot < slots, turns = slot < turning;
  const int ca = !live ? 0 : turns ? slot * V : p.R + 2 * V * (slot - turning), cb = !live ? 0 : turns ? half + slot * V : ca + V;
  const float inv_d = 1.0f / (float)p.D;
  float wa[V], wb[V], da[V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    wa[i] = live ? s.w[ca + i] : 0.f;
    wb[i] = live ? s.w[cb + i] : 0.f;
    da[i] = db[i] = 0.f;
  }
  const int chunks = (s.H + U - 1) / U;
  const long long items = (long long)p.B * p.L * chunks;
  // this group's items: first, first + step, ...; step = ((sb * L) + sl) * chunks + sc
  const long long first = (long long)blockIdx.x * per + g, step = (long long)s.blocks * per;
  const int sc = (int)(step % chunks), sl = (int)(step / chunks % p.L), sb = (int)(step / chunks / p.L);
  int c = (int)(first % chunks), l = (int)(first / chunks % p.L), b = (int)(first / chunks / p.L);
  for (long long item = first; item < items; item += step) {
    vec xa0[U], xb0[U], ya0[U], yb0[U];
    float cs[V], sn[V];
    const long long row = ((long long)b * p.L + l) * s.H + c * U;
    const int heads = live ? (s.H - c * U < U ? s.H - c * U : U) : 0;
    const T* x = (const T*)s.x + b * s.sb + l * s.sl + (long long)(c * U) * s.sh;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < heads) {
        xa0[u] = *(const vec*)(x + u * s.sh + ca);
        xb0[u] = *(const vec*)(x + u * s.sh + cb);
        if (BWD) {
          const T* dy = (const T*)s.dy + (row + u) * p.D;
          ya0[u] = *(const vec*)(dy + ca);
          yb0[u] = *(const vec*)(dy + cb);
        }
      }
    const long long at = turns ? angle_row(p, b, l) : -1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      cs[i] = at >= 0 ? p.cosv[at * half + ca + i] : turns ? __builtin_nanf("") : 1.f;
      sn[i] = at >= 0 ? p.sinv[at * half + ca + i] : turns ? __builtin_nanf("") : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = u < heads;
      float xa[V], xb[V], sq = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xa[i] = on ? (float)xa0[u][i] : 0.f;
        xb[i] = on ? (float)xb0[u][i] : 0.f;
        sq += xa[i] * xa[i] + xb[i] * xb[i];
      }
      sq = group_sum(sq, p.lanes);
      const float r = 1.0f / sqrtf(sq * inv_d + p.eps);
      T* y = (T*)s.y + (row + u) * p.D;
      vec oa, ob;
      if (!BWD) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float na = xa[i] * r * wa[i], nb = xb[i] * r * wb[i];
          oa[i] = (T)(turns ? na * cs[i] - nb * sn[i] : na);
          ob[i] = (T)(turns ? nb * cs[i] + na * sn[i] : nb);
        }
      } else {
        float ga[V], gb[V], dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float ya = on ? (float)ya0[u][i] : 0.f, yb = on ? (float)yb0[u][i] : 0.f;
          const float na = turns && on ? ya * cs[i] + yb * sn[i] : ya, nb = turns && on ? yb * cs[i] - ya * sn[i] : yb;
          xa[i] *= r;
          xb[i] *= r;
          da[i] += na * xa[i];
          db[i] += nb * xb[i];
          ga[i] = na * wa[i];
          gb[i] = nb * wb[i];
          dot += ga[i] * xa[i] + gb[i] * xb[i];
        }
        dot = group_sum(dot, p.lanes) * inv_d;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          oa[i] = (T)(r * (ga[i] - xa[i] * dot));
          ob[i] = (T)(r * (gb[i] - xb[i] * dot));
        }
      }
      if (on) {
        *(vec*)(y + ca) = oa;
        *(vec*)(y + cb) = ob;
      }
    }
    c += sc;
    l += sl;
    b += sb;
    if (c >= chunks) { c -= chunks; ++l; }
    if (l >= p.L) { l -= p.L; ++b; }
  }
  if (BWD) {
    // the block's sum of dw: each lane writes its own slots, then one thread per channel adds the row groups in order
    extern __shared__ float red[];                 // [per][D]
    if (live) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        red[g * p.D + ca + i] = da[i];
        red[g * p.D + cb + i] = db[i];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.D; c += 256) {
      float t = 0.f;
      for (int i = 0; i < per; ++i) t += red[i * p.D + c];
      s.part[(size_t)blockIdx.x * p.D + c] = t;
    }
  }
}

// dw[c] = sum over blocks of part[block][c]: 32 channels x 8 strided runs per block, joined in a fixed order
__global__ __launch_bounds__(256) void dw_final_k(const float* pq, int nq, float* dwq, const float* pk, int nk, float* dwk, int D) {
  __shared__ float red[8][33];
  const float* part = blockIdx.y ? pk : pq;
  const int n = blockIdx.y ? nk : nq, tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
  float t = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int i = ty; i < n; i += 8) t += part[(size_t)i * D + c];
  }
  red[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && c < D) {
    for (int i = 1; i < 8; ++i) t += red[i][tx];
    (blockIdx.y ? dwk : dwq)[c] = t;
  }
}

bool fits(const QkP& p, int V, int esize, bool bwd) {
  if ((p.R / 2) % V || (p.D - p.R) % (2 * V)) return false;
  const uintptr_t m = (uintptr_t)V * esize - 1;
  for (int i = 0; i < 2; ++i) {
    const Side& s = p.s[i];
    if ((s.sb % V) || (s.sl % V) || (s.sh % V) || (p.D % V)) return false;
    if ((((uintptr_t)s.x) | ((uintptr_t)s.y) | (bwd ? (uintptr_t)s.dy : 0)) & m) return false;
  }
  return true;
}

template <typename T, int V>
void launch(QkP& p, bool bwd, int nq, int nk, hipStream_t st) {
  const dim3 grid(nq > nk ? nq : nk, 2);
  if (bwd) hipLaunchKernelGGL((qk_norm_rotary_k<T, V, true, kHeadsBwd>), grid, dim3(256), (size_t)(256 / p.lanes) * p.D * 4, st, p);
  else hipLaunchKernelGGL((qk_norm_rotary_k<T, V, false, kHeadsFwd>), grid, dim3(256), 0, st, p);
}

// blocks of one side: a group of rows each, at most `most` (backward: each leaves a partial sum of dw)
int side_blocks(long long rows, int per, int most) {
  const long long n = (rows + per - 1) / per;
  return (int)(n < 1 ? 1 : n > most ? most : n);
}

int run(QkP& p, int dtype, bool bwd, float* dwq, float* dwk, float* ws, long long ws_floats, hipStream_t st) {
  if (p.B < 1 || p.L < 1 || p.s[0].H < 1 || p.s[1].H < 1 || p.D < 2 || (p.D & 1) || p.D > 128 || p.R < 0 || (p.R & 1) || p.R > p.D)
    return SO_ERR_SHAPE;
  if (!p.s[0].x || !p.s[1].x || !p.s[0].w || !p.s[1].w || (p.R && (!p.cosv || !p.sinv))) return SO_ERR_SHAPE;      // (an empty table has no address)
  if ((dtype != SO_F32 && dtype != SO_BF16) || (!p.pos && (p.start < 0 || p.start + p.L > p.P))) return SO_ERR_SHAPE;
  const int esize = dtype == SO_F32 ? 4 : 2;
  int V = 16 / esize;
  while (V > 1 && !fits(p, V, esize, bwd)) V >>= 1;
  if (V == 1 && !fits(p, 1, esize, bwd)) return SO_ERR_ALIGN;
  p.lanes = 1;
  while (p.lanes < p.D / (2 * V)) p.lanes <<= 1;
  const int per = 256 / p.lanes, u = bwd ? kHeadsBwd : kHeadsFwd;
  for (int i = 0; i < 2; ++i) p.s[i].blocks = side_blocks((long long)p.B * p.L * ((p.s[i].H + u - 1) / u), per, bwd ? kBlocksBwd : 1 << 20);
  if (bwd) {
    if (ws_floats < (long long)(p.s[0].blocks + p.s[1].blocks) * p.D) return SO_ERR_SHAPE;
    p.s[0].part = ws;
    p.s[1].part = ws + (size_t)p.s[0].blocks * p.D;
  }
  const int nq = p.s[0].blocks, nk = p.s[1].blocks;
  if (dtype == SO_F32) {
    if (V == 4) launch<float, 4>(p, bwd, nq, nk, st);
    else if (V == 2) launch<float, 2>(p, bwd, nq, nk, st);
    else launch<float, 1>(p, bwd, nq, nk, st);
  } else {
    if (V == 8) launch<__bf16, 8>(p, bwd, nq, nk, st);
    else if (V == 4) launch<__bf16, 4>(p, bwd, nq, nk, st);
    else if (V == 2) launch<__bf16, 2>(p, bwd, nq, nk, st);
    else launch<__bf16, 1>(p, bwd, nq, nk, st);
  }
  int err = SO_LAUNCH_CHECK();
  if (err || !bwd) return err;
  hipLaunchKernelGGL(dw_final_k, dim3((p.D + 31) / 32, 2), dim3(256), 0, st, p.s[0].part, nq, dwq, p.s[1].part, nk, dwk, p.D);
  return SO_LAUNCH_CHECK();
}

QkP make(const so_qk_desc& d) {
  QkP p = {};
  p.s[0].x = d.q; p.s[0].sb = d.sqb; p.s[0].sl = d.sql; p.s[0].sh = d.sqh; p.s[0].H = d.Hq; p.s[0].w = d.wq;
  p.s[1].x = d.k; p.s[1].sb = d.skb; p.s[1].sl = d.skl; p.s[1].sh = d.skh; p.s[1].H = d.Hk; p.s[1].w = d.wk;
  p.cosv = d.cosv; p.sinv = d.sinv; p.P = d.P; p.pos = d.pos; p.pos64 = d.pos64; p.pos_sb = d.pos_sb; p.pos_sl = d.pos_sl; p.start = d.start;
  p.B = d.B; p.L = d.L; p.D = d.D; p.R = d.R; p.eps = d.eps;
  return p;
}

}  // namespace

extern "C" {

int so_qk_desc_bytes(void) { return (int)sizeof(so_qk_desc); }

int so_qk_norm_rotary_fwd(const void* desc, void* yq, void* yk, void* stream) {
  if (!desc || !yq || !yk) return SO_ERR_SHAPE;
  const so_qk_desc& d = *(const so_qk_desc*)desc;
  QkP p = make(d);
  p.s[0].y = yq;
  p.s[1].y = yk;
  return run(p, d.dtype, false, nullptr, nullptr, nullptr, 0, (hipStream_t)stream);
}

long long so_qk_norm_rotary_ws_floats(int D) { return 2LL * kBlocksBwd * D; }

int so_qk_norm_rotary_bwd(const void* desc, const void* dyq, const void* dyk, void* dq, void* dk, float* dwq, float* dwk, float* ws,
                          long long ws_floats, void* stream) {
  if (!desc || !dyq || !dyk || !dq || !dk || !dwq || !dwk || !ws) return SO_ERR_SHAPE;
  const so_qk_desc& d = *(const so_qk_desc*)desc;
  QkP p = make(d);
  p.s[0].y = dq; p.s[0].dy = dyq;
  p.s[1].y = dk; p.s[1].dy = dyk;
  return run(p, d.dtype, true, dwq, dwk, ws, ws_floats, (hipStream_t)stream);
}

}  // extern "C"
