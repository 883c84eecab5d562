// Shared pieces of the multi-head attention kernels (mha_fwd.hip, mha_bwd.hip), gfx950.
//
// One 16-byte fragment per lane is the unit of all products: bf16 holds 8 values of it (one v_mfma_f32_32x32x16_bf16: lane (row l %
// 32, half l / 32) supplies k = 8 half + e), fp32 holds 4 (four v_mfma_f32_32x32x2_f32: MFMA e takes k = 4 half + e).  Either way a
// product step covers 32 bytes of the k axis and the byte addresses are the same for both types.
//
// A 32 x 32 accumulator holds, in lane (column l % 32, half), register r: row (r & 3) + 8 (r >> 2) + 4 half.  The rows of a score
// product are dealt out so that this is tile row 16 half + r (tile_row: lane l of the A fragment reads tile row tile_row(l)): a lane
// then holds sixteen CONSECUTIVE rows.  Scores are computed TRANSPOSED against what they multiply next (rows = the axis that the next
// product sums over), so registers 4 c .. 4 c + 3 (fp32) or 8 c .. 8 c + 7 (bf16) are already the B fragment of that product's step c:
//     row(step c, element e) = 16 half + 4 c + e (fp32)  or  16 half + 8 c + e (bf16);
// its A fragment is read to match: single dwords (fp32) or two ds_read_b64_tr_b16 (bf16), which transpose on the way.  The products
// whose rows are channels keep the plain order.
#pragma once
#include <hip/hip_runtime.h>
#include "common.h"
#include "../../include/shineon_hip.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // four floats at any float's address

namespace mha {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int E = 4;          // elements of a 16-byte fragment
  typedef f32x4 frag;
};
template <> struct Elem<__bf16> {
  static constexpr int E = 8;
  typedef bf16x8 frag;
};

__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}

__device__ __forceinline__ int acc_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }
__device__ __forceinline__ int tile_row(int l) { return 16 * ((l >> 2) & 1) + 4 * (l >> 3) + (l & 3); }

template <int N> struct Log2 { static constexpr int v = 1 + Log2<N / 2>::v; };
template <> struct Log2<1> { static constexpr int v = 0; };

// A tile of rows in LDS: DP channels of T per row as 16-byte chunks, chunk c of row r at position c ^ f(r); rows are a power of two
// chunks long.  f makes both ways of reading free of bank conflicts (64 banks; 16 lanes of a ds_read_b128 go together, those whose lane
// bits 2, 3, 4 have the same parity): in row_frag these 16 lanes hold all values of row bits 0 - 3, in col_frag four rows of row bits
// 0 - 1 are read in four neighbouring chunks, and an fp32 dword read takes two rows 16 apart.
template <typename T, int DP>
struct Tile {
  static constexpr int E = Elem<T>::E, NC = DP / E;                      // chunks that hold data
  static constexpr int NP = NC <= 4 ? 4 : NC <= 8 ? 8 : NC <= 16 ? 16 : 32;   // chunks of a row in LDS
  static constexpr int kRowBytes = NP * 16;
  __device__ static __forceinline__ int swz(int row) {
    const int hi = (row >> 2) & 3;
    return NP == 4 ? hi : NP == 8 ? hi | ((row & 2) << 1) : (hi | ((row & 3) << 2)) ^ ((row >> 1) & 8);
  }
  __device__ static __forceinline__ int at(int row, int chunk) { return row * kRowBytes + ((chunk ^ swz(row)) << 4); }
};

// LDS by byte address, so that constants end up in the offset field of the instruction
typedef __attribute__((address_space(3))) char* lds_ptr;
__device__ __forceinline__ int lds_at(const char* p) { return __builtin_amdgcn_readfirstlane((int)(unsigned)(unsigned long long)(lds_ptr)p); }
template <typename V>
__device__ __forceinline__ V lds_read(int at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) V*>((unsigned)at);
}

// A branch whose condition is the same for the whole block and rarely true: keeps hipcc from computing both sides
__device__ __forceinline__ void seldom() { asm volatile("; seldom"); }

// Fragment addresses.  The swizzle is an XOR of address bits, so every fragment of a tile is (lane's base ^ constant) + constant; tiles
// start at multiples of 512 bytes.  The base is made opaque at every use: otherwise hipcc keeps the two dozen addresses of a tile in
// registers over the whole loop, and spills.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
// Values that must have arrived here: hipcc puts its wait for a load in front of the first use, and where that is inside a loop the wait
// (vmcnt 0) comes in every iteration and covers the fills in flight
template <typename V>
__device__ __forceinline__ void settle(V& x) {
  asm volatile("" : "+v"(x));
}
template <typename T, int DP>
struct Reader {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::frag frag;
  int rows, cols;      // byte addresses of the lane's row and column fragments in a tile at sm
  __device__ __forceinline__ Reader(const char* sm, int lane) {
    const int half = lane >> 5, li = lane & 31;
    rows = lds_at(sm) + TL::at(tile_row(li), half);
    if constexpr (sizeof(T) == 4) cols = lds_at(sm) + TL::at(16 * half, li >> 2) + 4 * (li & 3);
    else cols = lds_at(sm) + TL::at(16 * half + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
  }
  // A fragment: row tile_row(lane) of the 32 rows at byte `at` of a tile, step m of the channel axis
  __device__ __forceinline__ frag row(int base, int m, int at) const { return lds_read<frag>((base ^ (m << 5)) + at); }
  // A fragment: column 32 t + lane, step c of the row axis of the 32 rows at byte `at`
  __device__ __forceinline__ frag col(int base, int t, int c, int at) const {
    if constexpr (sizeof(T) == 4) {
      frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = lds_read<float>((base ^ (((8 * t) ^ TL::swz(4 * c + e)) << 4)) + at + (4 * c + e) * TL::kRowBytes);
      return f;
    } else {
      typedef __attribute__((address_space(3))) s16x4* lds_p;
      union { s16x4 s[2]; frag f; } u;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        u.s[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_p)(unsigned)((base ^ (((4 * t) ^ TL::swz(8 * c + 4 * i)) << 4)) + at + (8 * c + 4 * i) * TL::kRowBytes));
      return u.f;
    }
  }
};

// sixteen consecutive floats at a byte address that is a multiple of 4
__device__ __forceinline__ void lds_read16(int at, f32x16& v) {
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = lds_read<float>(at + 4 * r);
}

// accumulator registers of step c as a B fragment; bf16 rounds here (half a step, 2^-8 of the value: the products run at the rate of
// 16-bit operands; sums, statistics and accumulators stay fp32).  The backward pass takes one fragment, the forward pass as many as the
// value has bits (kPieces)
__device__ __forceinline__ void to_frag(const f32x16& a, int c, f32x4& f) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = a[4 * c + e];
}
__device__ __forceinline__ void to_frag(const f32x16& a, int c, bf16x8& f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (__bf16)a[8 * c + e];
}

// One product phase of N steps: step m multiplies with the fragment that was requested N steps ago and requests the one for step m of
// the next phase into its place.  The order is pinned (sched_barrier): left to itself hipcc reads each fragment right before its MFMA and
// exposes the LDS latency at every step.
template <int N, typename F, typename Use, typename Next>
__device__ __forceinline__ void phase(F (&buf)[N], Use use, Next next) {
#pragma unroll
  for (int m = 0; m < N; ++m) {
    use(m, buf[m]);
    buf[m] = next(m);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <int N, typename F, typename Use>
__device__ __forceinline__ void last_phase(F (&buf)[N], Use use) {
#pragma unroll
  for (int m = 0; m < N; ++m) use(m, buf[m]);
}

// 16-byte chunk of a row in global memory, zero when `on` is false (the address is then not formed)
template <typename T>
__device__ __forceinline__ f32x4 load_chunk(const T* row, int chunk, bool on) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (on) v = *reinterpret_cast<const f32x4*>(row + chunk * Elem<T>::E);
  return v;
}
template <typename T>
__device__ __forceinline__ typename Elem<T>::frag as_frag(f32x4 v) {
  union { f32x4 v; typename Elem<T>::frag f; } u;
  u.v = v;
  return u.f;
}

// Fills a tile of ROWS rows in LDS from rows `stride` bytes apart, by LDS-DMA (no registers, no ds_write).  A fill writes lane after
// lane, so the chunk swizzle is applied on the source side.  Rows whose bit is clear and channels behind D are requested at an offset
// outside the descriptor and arrive as zeros; nothing outside the operand is read.  The caller drains before the barrier that publishes
// the tile.
//
// The fills are written in assembly so that hipcc does not know of them: it makes every ds_read_b64_tr wait for all fills in flight
// (vmcnt 0), and the tile after the current one would arrive with its full latency exposed.  They have no register results; s_nop 4
// covers a descriptor that a vector instruction (v_readfirstlane) has just written, which hipcc does not see to in assembly; drain()
// is the wait that a barrier needs in front of it.  An own wait of hipcc's for its loads can only become longer by them.
__device__ __forceinline__ i32x4 rsrc_of(const void* base, unsigned bytes) {      // raw buffer over [base, base + bytes)
  const unsigned long long a = (unsigned long long)base;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)a), __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32) & 0xFFFF),
               __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
__device__ __forceinline__ void dma16(i32x4 rsrc, int lds, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ void dma4(i32x4 rsrc, int lds, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}
// all but the N youngest requests of the wave have arrived
template <int N>
__device__ __forceinline__ void arrived() {
  static_assert(N < 64, "six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// the wave's LDS reads so far are in registers: what they read may be overwritten
__device__ __forceinline__ void lds_done() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ void drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <typename T, int DP, int ROWS, int WAVES>
struct Filler {
  typedef Tile<T, DP> TL;
  static constexpr int N = ROWS * TL::NP / (64 * WAVES), RPF = 64 * WAVES / TL::NP;   // fills per thread; rows per round of fills
  static_assert(N * 64 * WAVES == ROWS * TL::NP, "whole fills");
  unsigned off[N];
  int row0;
  __device__ __forceinline__ Filler(int D, unsigned stride, int tid) {
    row0 = tid / TL::NP;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int row = row0 + j * RPF, ch = (tid & (TL::NP - 1)) ^ TL::swz(row);
      off[j] = ch * TL::E < D ? row * stride + ch * 16 : 0x80000000u;
    }
  }
  // rows [base_row, base_row + ROWS) of the tile at `src`; bits: one per row (64 rows from base_row 0, further ones in `more`)
  __device__ __forceinline__ void fill(char* tile, const void* src, unsigned long long bits, unsigned long long more, int wave) const {
    const i32x4 r = rsrc_of(src, 0x7FFFFFFFu);
    const int at = lds_at(tile) + wave * 1024;
    const bool all = bits == ~0ULL && (ROWS <= 64 || more == ~0ULL);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      unsigned o = off[j];
      if (!all) {
        const int row = row0 + j * RPF;
        const unsigned long long w = ROWS > 64 && row >= 64 ? more : bits;
        o = (w >> (row & 63)) & 1 ? o : 0x80000000u;
      }
      dma16(r, at + j * WAVES * 1024, o);
    }
  }
};

// n dwords of global memory -> LDS, by LDS-DMA; wave w of `WAVES` takes the 64-dword pieces w, w + WAVES, ...  `bytes` bounds the source
// (what lies behind arrives as zeros).  LDS is written in whole pieces.
template <int WAVES>
__device__ __forceinline__ void fill_dwords(void* dst, const void* src, int n, unsigned bytes, int wave, int lane) {
  const i32x4 r = rsrc_of(src, bytes);
  const int at = lds_at((const char*)dst);
  for (int i = 64 * wave; i < n; i += 64 * WAVES)
    dma4(r, at + 4 * i, 4 * (i + lane));
}

// sum / maximum over the two halves of a wave, without LDS
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// visible keys [64 w, 64 w + 64) of a sample as bits; keys behind the last are invisible
__device__ __forceinline__ unsigned long long tail_word(int w, int Lk) {
  const int left = Lk - 64 * w;
  return left >= 64 ? ~0ULL : left <= 0 ? 0ULL : (1ULL << left) - 1;
}
// Mask words of an ascending walk: the wave holds 64 of them, one per lane, and hands them out as scalars.
struct KeyWords {
  const unsigned long long* words;
  int n, Lk, first, lane;
  unsigned long long mine;
  __device__ __forceinline__ KeyWords(const unsigned long long* words, int n, int Lk, int lane)
      : words(words), n(n), Lk(Lk), first(-64), lane(lane), mine(0) {}
  __device__ __forceinline__ unsigned long long get(int w) {
    const unsigned long long tail = tail_word(w, Lk);
    if (!words) return tail;
    if (w < first || w >= first + 64) {
      first = w;
      mine = w + lane < n ? words[w + lane] : 0ULL;
      settle(mine);
    }
    const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)mine, w - first), hi = __builtin_amdgcn_readlane((int)(unsigned)(mine >> 32), w - first);
    return tail & (((unsigned long long)hi << 32) | lo);
  }
};

// first and one-past-last word with a visible key (the whole wave calls it)
__device__ __forceinline__ void word_range(const unsigned long long* words, int Lk, int lane, int& lo, int& hi) {
  const int n = (Lk + 63) >> 6;
  lo = 0;
  hi = n;
  if (!words) return;
  lo = n;
  hi = 0;
  // eight words per lane at a time, so that a long row costs one latency per 32768 keys
  for (int w0 = 0; w0 < n; w0 += 512) {
    unsigned long long x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int w = w0 + 64 * j + lane;
      x[j] = words[w < n ? w : n - 1];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned long long any = __ballot(w0 + 64 * j + lane < n && x[j] != 0);
      if (any) {
        if (lo == n) lo = w0 + 64 * j + __builtin_ctzll(any);
        hi = w0 + 64 * j + 64 - __builtin_clzll(any);
      }
    }
  }
}

// 2^x for the softmax: v_exp_f32 (1 ulp); x <= 0 here up to rounding, results below 2^-126 vanish
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// most codes between the first and last of n consecutive tokens of a map with rows of `width` (a sequence: 1)
__host__ __device__ inline int code_span(int n, int width) {
  return n < 2 ? 0 : (n - 1) + ((n - 2) / width + 1) * (width - 1);
}

// Block -> (sample, key head, block of that group).  A one-dimensional grid; XCD x = id % 8 gets the x-th contiguous eighth of an order
// in which the blocks of a (sample, key head), which read the same keys and values, follow each other: they stay in that XCD's L2
// (4 MB: 8192 keys and values of 128 bf16 channels).  The order goes through half of every group's blocks and then through the other
// half, samples innermost, so that an XCD meets several samples of a ragged batch.
struct BlockOf { int b, hk, idx; };
__device__ __forceinline__ BlockOf block_of(int B, int Hk, int per) {
  const unsigned total = gridDim.x, x = blockIdx.x & 7, each = total >> 3, rest = total & 7;
  unsigned v = x * each + (x < rest ? x : rest) + (blockIdx.x >> 3);
  const unsigned groups = B * Hk, first = (per + 1) >> 1;
  unsigned g, idx;
  if (v < groups * first) {
    g = v / first;
    idx = v - g * first;
  } else {
    v -= groups * first;
    const unsigned second = per - first;
    g = v / second;
    idx = first + v - g * second;
  }
  return BlockOf{(int)(g % B), (int)(g / B), (int)idx};
}

}  // namespace mha

int so_mha_check(const so_mha_desc* d);   // shape, type and alignment rules that all entry points share

// 128-row tiles in n rows; the last pays for its 32-row waves only
double mha_tiles(int n);
// Parts that the sum axis of a kernel is cut into (at most 8, at most `most`): blocks on one CU share its pipes, so a pass takes as long as
// the CU with most blocks, ceil(blocks parts / 256) / parts of a whole block's `block_us`; joining costs join_us and, for every part, writing and
// reading `part_bytes` (both counted) at `rate` bytes per us - at most that of a large copy where the parts together outgrow the caches.  More
// parts are taken when they bring the estimate below `gain` of the last choice.
int mha_split_parts(double blocks, double block_us, double join_us, double part_bytes, double rate, int most, double gain);
// block_us from a block's FLOP: what a CU reaches in these kernels
inline double mha_us(double flop, int dtype) { return flop / (dtype == SO_F32 ? 0.45e6 : 3.0e6); }
