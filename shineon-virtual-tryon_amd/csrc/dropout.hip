// Dropout whose mask is a function of a counter and is never stored, gfx950.
//
//   y[e] = residual[e] + (keep(e) ? x[e] * scale : 0),   keep(e) = word (e mod 4) of philox(seed, offset + e div 4) >= threshold
//
// with e the element's number in row-major order (channels innermost for an NHWC map, whatever its pitch), threshold =
// round(p 2^32) and scale = 1 / (1 - p).  The backward pass is the same kernel on dy.  seed and offset are read from DEVICE memory,
// so a captured graph draws a new mask at every replay (so_rng_draw is the node that moves the counter on).
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64
// bit products, 64 key bits, here 64 counter bits and 64 zero bits.  One block of four words serves four elements.
#include "common.h"
#include "../../include/shineon_hip.h"

namespace {

struct Words { unsigned w[4]; };

__device__ __forceinline__ Words philox(unsigned long long seed, unsigned long long ctr) {
  unsigned c0 = (unsigned)ctr, c1 = (unsigned)(ctr >> 32), c2 = 0, c3 = 0;
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
    c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
    c1 = (unsigned)p1;
    c3 = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

template <typename T> struct Pack;
template <> struct Pack<float> { static constexpr int kVec = 4; typedef f32x4 vec; };
template <> struct Pack<__bf16> { static constexpr int kVec = 8; typedef __bf16 vec __attribute__((ext_vector_type(8))); };

struct DropP {
  const void* x;
  const void* res;
  void* y;
  const long long* rng;
  long long n, C, ldx, ldr, ldy;   // elements; row length and pitches
  unsigned long long threshold;    // 0 .. 2^32
  float scale;
};

// Bound by HBM: the ten rounds take less than the loads.  8 x 4099 x 1024, bf16: 39-42 us with a residual (4.8-5.1 TB/s), 23 us without (5.7).
// Eight elements (two generator blocks) per thread, so that a bf16 thread moves 16 bytes.  VEC: dense operands, 16-byte aligned; otherwise every
// element is addressed by its row and column, and a wave's accesses are 16 or 32 bytes apart: with rows 2048 apart or one element off alignment
// 112-114 us with a residual (1.8 TB/s), fp32 427 us (0.94 TB/s).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_k(const DropP p) {
  const long long e0 = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e0 >= p.n) return;
  const unsigned long long seed = (unsigned long long)p.rng[0], ctr = (unsigned long long)p.rng[1] + (unsigned long long)(e0 >> 2);
  const T* x = (const T*)p.x;
  const T* res = (const T*)p.res;
  T* y = (T*)p.y;
  if (VEC && e0 + 8 <= p.n) {
    constexpr int KV = Pack<T>::kVec, NV = 8 / KV;
    typedef typename Pack<T>::vec vec;
    vec v[NV], r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = *(const vec*)(x + e0 + i * KV);
    if (res) {
#pragma unroll
      for (int i = 0; i < NV; ++i) r[i] = *(const vec*)(res + e0 + i * KV);
    }
    const Words w[2] = {philox(seed, ctr), philox(seed, ctr + 1)};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < KV; ++j) {
        const int e = i * KV + j;
        float o = (unsigned long long)w[e >> 2].w[e & 3] >= p.threshold ? (float)v[i][j] * p.scale : 0.f;
        if (res) o += (float)r[i][j];
        v[i][j] = (T)o;
      }
      *(vec*)(y + e0 + i * KV) = v[i];
    }
    return;
  }
  const Words w[2] = {philox(seed, ctr), philox(seed, ctr + 1)};
  long long row = e0 / p.C, col = e0 - row * p.C;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e0 + e >= p.n) return;
    float o = (unsigned long long)w[e >> 2].w[e & 3] >= p.threshold ? (float)x[row * p.ldx + col] * p.scale : 0.f;
    if (res) o += (float)res[row * p.ldr + col];
    y[row * p.ldy + col] = (T)o;
    if (++col == p.C) { col = 0; ++row; }
  }
}

__global__ void rng_draw_k(long long* state, long long* out, long long blocks) {
  const long long seed = state[0], at = state[1];
  out[0] = seed;
  out[1] = at;
  state[1] = (long long)((unsigned long long)at + (unsigned long long)blocks);
}

template <typename T>
void launch(const DropP& p, bool vec, hipStream_t st) {
  const dim3 grid((unsigned)((p.n + 2047) / 2048));
  if (vec) hipLaunchKernelGGL((dropout_k<T, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((dropout_k<T, false>), grid, dim3(256), 0, st, p);
}

}  // namespace

extern "C" {

int so_rng_draw(void* state, void* out, long long blocks, void* stream) {
  if (!state || !out || blocks < 0) return SO_ERR_SHAPE;
  hipLaunchKernelGGL(rng_draw_k, dim3(1), dim3(1), 0, (hipStream_t)stream, (long long*)state, (long long*)out, blocks);
  return SO_LAUNCH_CHECK();
}

int so_dropout(int dtype, const void* x, long long ldx, const void* residual, long long ldr, void* y, long long ldy, long long rows,
               long long C, const void* rng, long long threshold, float scale, void* stream) {
  if ((dtype != SO_F32 && dtype != SO_BF16) || rows < 0 || C < 0 || ldx < C || ldy < C || (residual && ldr < C)) return SO_ERR_SHAPE;
  if (threshold < 0 || threshold > (1LL << 32)) return SO_ERR_SHAPE;
  if (C && rows > (1LL << 40) / C) return SO_ERR_SHAPE;      // the grid's 2^31 blocks of 2048 elements
  if (rows == 0 || C == 0) return 0;
  if (!x || !y || !rng) return SO_ERR_SHAPE;
  DropP p = {};
  p.x = x; p.res = residual; p.y = y; p.rng = (const long long*)rng;
  p.n = rows * C; p.C = C; p.ldx = ldx; p.ldr = ldr; p.ldy = ldy;
  p.threshold = (unsigned long long)threshold; p.scale = scale;
  const bool dense = rows == 1 || (ldx == C && ldy == C && (!residual || ldr == C));
  const bool vec = dense && !((((uintptr_t)x) | ((uintptr_t)y) | ((uintptr_t)residual)) & 15);
  if (dtype == SO_F32) launch<float>(p, vec, (hipStream_t)stream);
  else launch<__bf16>(p, vec, (hipStream_t)stream);
  return SO_LAUNCH_CHECK();
}

}  // extern "C"
