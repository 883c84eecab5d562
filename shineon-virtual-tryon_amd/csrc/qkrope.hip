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

template <typename T, int V, bool BWD>
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
  const long long rows = (long long)p.B * p.L * s.H;
  for (long long row = (long long)blockIdx.x * per + g; row < rows; row += (long long)s.blocks * per) {
    const long long tok = row / s.H;
    const int h = (int)(row - tok * s.H), b = (int)(tok / p.L), l = (int)(tok - (long long)b * p.L);
    const T* x = (const T*)s.x + b * s.sb + l * s.sl + h * s.sh;
    float xa[V], xb[V], cs[V], sn[V], sq = 0.f;
    if (live) {
      const vec a = *(const vec*)(x + ca), bb = *(const vec*)(x + cb);
      long long at = turns ? angle_row(p, b, l) : 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        cs[i] = turns ? (at < 0 ? __builtin_nanf("") : p.cosv[at * half + ca + i]) : 1.f;
        sn[i] = turns ? (at < 0 ? __builtin_nanf("") : p.sinv[at * half + ca + i]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xa[i] = (float)a[i];
        xb[i] = (float)bb[i];
        sq += xa[i] * xa[i] + xb[i] * xb[i];
      }
    }
    sq = group_sum(sq, p.lanes);
    const float r = 1.0f / sqrtf(sq * inv_d + p.eps);
    T* y = (T*)s.y + row * p.D;
    if (!BWD) {
      if (live) {
        vec a, bb;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float na = xa[i] * r * wa[i], nb = xb[i] * r * wb[i];
          a[i] = (T)(turns ? na * cs[i] - nb * sn[i] : na);
          bb[i] = (T)(turns ? nb * cs[i] + na * sn[i] : nb);
        }
        *(vec*)(y + ca) = a;
        *(vec*)(y + cb) = bb;
      }
    } else {
      const T* dy = (const T*)s.dy + row * p.D;
      float ga[V], gb[V], dot = 0.f;
      if (live) {
        const vec a = *(const vec*)(dy + ca), bb = *(const vec*)(dy + cb);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float ya = (float)a[i], yb = (float)bb[i];
          const float na = turns ? ya * cs[i] + yb * sn[i] : ya, nb = turns ? yb * cs[i] - ya * sn[i] : yb;
          xa[i] *= r;
          xb[i] *= r;
          da[i] += na * xa[i];
          db[i] += nb * xb[i];
          ga[i] = na * wa[i];
          gb[i] = nb * wb[i];
          dot += ga[i] * xa[i] + gb[i] * xb[i];
        }
      }
      dot = group_sum(dot, p.lanes) * inv_d;
      if (live) {
        vec a, bb;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a[i] = (T)(r * (ga[i] - xa[i] * dot));
          bb[i] = (T)(r * (gb[i] - xb[i] * dot));
        }
        *(vec*)(y + ca) = a;
        *(vec*)(y + cb) = bb;
      }
    }
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
  if (bwd) hipLaunchKernelGGL((qk_norm_rotary_k<T, V, true>), grid, dim3(256), (size_t)(256 / p.lanes) * p.D * 4, st, p);
  else hipLaunchKernelGGL((qk_norm_rotary_k<T, V, false>), grid, dim3(256), 0, st, p);
}

// blocks of one side: enough to fill the chip eight blocks deep, never more than there are groups of rows
int side_blocks(long long rows, int per) {
  const long long n = (rows + per - 1) / per;
  return (int)(n < 1 ? 1 : n > 1024 ? 1024 : n);
}

int run(QkP& p, int dtype, bool bwd, float* dwq, float* dwk, float* ws, long long ws_floats, hipStream_t st) {
  if (p.B < 0 || p.L < 0 || p.s[0].H < 1 || p.s[1].H < 1 || p.D < 2 || (p.D & 1) || p.D > 128 || p.R < 0 || (p.R & 1) || p.R > p.D)
    return SO_ERR_SHAPE;
  if ((dtype != SO_F32 && dtype != SO_BF16) || (!p.pos && (p.start < 0 || p.start + p.L > p.P))) return SO_ERR_SHAPE;
  const int esize = dtype == SO_F32 ? 4 : 2;
  int V = 16 / esize;
  while (V > 1 && !fits(p, V, esize, bwd)) V >>= 1;
  if (V == 1 && !fits(p, 1, esize, bwd)) return SO_ERR_ALIGN;
  p.lanes = 1;
  while (p.lanes < p.D / (2 * V)) p.lanes <<= 1;
  const int per = 256 / p.lanes;
  for (int i = 0; i < 2; ++i) p.s[i].blocks = side_blocks((long long)p.B * p.L * p.s[i].H, per);
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

QkP make(const void* q, long long sqb, long long sql, long long sqh, int Hq, const void* k, long long skb, long long skl,
         long long skh, int Hk, const float* wq, const float* wk, const float* cosv, const float* sinv, long long P, const void* pos,
         int pos64, long long pos_sb, long long pos_sl, long long start, int B, int L, int D, int R, float eps) {
  QkP p = {};
  p.s[0].x = q; p.s[0].sb = sqb; p.s[0].sl = sql; p.s[0].sh = sqh; p.s[0].H = Hq; p.s[0].w = wq;
  p.s[1].x = k; p.s[1].sb = skb; p.s[1].sl = skl; p.s[1].sh = skh; p.s[1].H = Hk; p.s[1].w = wk;
  p.cosv = cosv; p.sinv = sinv; p.P = P; p.pos = pos; p.pos64 = pos64; p.pos_sb = pos_sb; p.pos_sl = pos_sl; p.start = start;
  p.B = B; p.L = L; p.D = D; p.R = R; p.eps = eps;
  return p;
}

}  // namespace

extern "C" {

int so_qk_norm_rotary_fwd(int dtype, const void* q, long long sqb, long long sql, long long sqh, int Hq, const void* k, long long skb,
                          long long skl, long long skh, int Hk, const float* wq, const float* wk, const float* cosv,
                          const float* sinv, long long P, const void* pos, int pos64, long long pos_sb, long long pos_sl,
                          long long start, void* yq, void* yk, int B, int L, int D, int R, float eps, void* stream) {
  QkP p = make(q, sqb, sql, sqh, Hq, k, skb, skl, skh, Hk, wq, wk, cosv, sinv, P, pos, pos64, pos_sb, pos_sl, start, B, L, D, R, eps);
  p.s[0].y = yq;
  p.s[1].y = yk;
  return run(p, dtype, false, nullptr, nullptr, nullptr, 0, (hipStream_t)stream);
}

long long so_qk_norm_rotary_ws_floats(int D) { return 2LL * 1024 * D; }

int so_qk_norm_rotary_bwd(int dtype, const void* q, long long sqb, long long sql, long long sqh, int Hq, const void* k, long long skb,
                          long long skl, long long skh, int Hk, const float* wq, const float* wk, const float* cosv,
                          const float* sinv, long long P, const void* pos, int pos64, long long pos_sb, long long pos_sl,
                          long long start, const void* dyq, const void* dyk, void* dq, void* dk, float* dwq, float* dwk, int B, int L,
                          int D, int R, float eps, float* ws, long long ws_floats, void* stream) {
  QkP p = make(q, sqb, sql, sqh, Hq, k, skb, skl, skh, Hk, wq, wk, cosv, sinv, P, pos, pos64, pos_sb, pos_sl, start, B, L, D, R, eps);
  p.s[0].y = dq; p.s[0].dy = dyq;
  p.s[1].y = dk; p.s[1].dy = dyk;
  return run(p, dtype, true, dwq, dwk, ws, ws_floats, (hipStream_t)stream);
}

}  // extern "C"
