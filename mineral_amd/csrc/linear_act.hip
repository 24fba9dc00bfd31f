// Linear layer with bias, activation and residual in its epilogue for gfx950, and its gradient:
//   z = x W^T + b, y = act(z) + residual;   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum dz
// One tiled product D[m][n] = sum_r A(m, r) B(n, r) serves the three: an operand lies with the reduction index along its rows (x and
// W forward, dz for dx) or with rows of the reduction index (W for dx, both for dW), and goes to LDS as it lies; fragments of the
// first kind are 16-byte reads, of the second transposing reads.  Tiles of 16-bit operands whose rows lie on 16-byte addresses go
// straight to LDS, several steps ahead of the MFMAs; others travel through registers one step ahead.
// The MFMAs take the operands swapped, so a lane's accumulators are four neighbouring columns of one row; the epilogue passes them
// through LDS once and then works on rows: bias, activation and its slope, residual and stores in 16-byte units.
// fp32 operands are split exactly into three bf16 terms on their way to LDS and multiply in six products, smallest first.
// dW sums over all rows: they are split over blocks whose partial sums are added in a fixed order.
// Bound: 32768 rows, 512 -> 2048, bf16, SiLU, residual: forward 165 us (435 MB to move and 69 GFLOP; the epilogue's loads and stores
// beside products of 16 steps only), dz 88 us (403 MB, 4.6 TB/s), dx 84 us (818 TFLOP/s), dW 95 + 7 us (723 TFLOP/s); plain products
// of this shape by the library run at 759.  8192^3: dW 1.07 PFLOP/s.  fp32, 512 -> 256, ELU: 53 us, 6 x 161 TFLOP/s of bf16 products.
#include "memory_common.hip.h"

#include <type_traits>

using namespace mrl::mem;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

enum { LAY_K = 0, LAY_R = 1 };   // reduction index along the rows / rows of the reduction index

struct MmP {
  const void *a, *b;
  int64_t lda, ldb;
  int M, N;                 // rows of D (A's), columns (B's)
  int64_t R;                // reduction length
  int64_t r_split;          // reduction length of a split (a multiple of the step)
  int m_tiles, n_tiles, blocks;
  void* y;                  // [M][N]
  float* slab;              // instead of y: [splits][M][N] fp32
  const void *bias, *residual;
  void* slope;              // act'(z): fp32, or packed to 16 bits beside 16-bit types
  int act;
  float gain;               // of a gradient's products beside fp16 (a power of two)
};

// one 16-byte unit, elements beyond `left` zero; addresses need only the element's alignment
template <typename T> __device__ __forceinline__ u32x4 load_unit(const T* p, int64_t left) {
  constexpr int E = 16 / (int)sizeof(T);
  u32x4 w = {0u, 0u, 0u, 0u};
  if (left >= E) __builtin_memcpy(&w, p, 16);
  else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) {
        if constexpr (sizeof(T) == 4) w[e] = __builtin_bit_cast(unsigned, p[e]);
        else w[e / 2] |= (unsigned)__builtin_bit_cast(unsigned short, p[e]) << (16 * (e & 1));
      }
  }
  return w;
}

template <typename T> struct Frag;
template <> struct Frag<__bf16> {
  static constexpr int NP = 1;
  typedef bf16x8 F;
  static __device__ __forceinline__ f32x16 mul(const F& a, const F& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<_Float16> {
  static constexpr int NP = 1;
  typedef f16x8 F;
  static __device__ __forceinline__ f32x16 mul(const F& a, const F& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<float> {
  static constexpr int NP = 3;
  typedef bf16x8 F;
  static __device__ __forceinline__ f32x16 mul(const F& a, const F& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// One operand's tile of a step: ROWS rows (of A or B) x BK reduction indices, as lines of WIDTH elements.
// LAY_K lines outside the matrix repeat its last one and columns beyond its edge hold what lies there: they only reach outputs that are
// not stored.  Reduction indices beyond the end read as zero in both operands.  A step that is whole and touches nothing beyond the
// matrix's last element (`whole`) is loaded without checks, the others element by element where a 16-byte unit is cut.
// DIRECT: rows are whole 16-byte units on 16-byte addresses; the loads write LDS themselves (no registers, the next stage is in
// flight during a whole step), which fixes the lines' pitch, so the 16-byte pieces of a line are permuted by its number instead to
// spread the fragment reads over the banks.
template <typename T, int LAY, int ROWS, int BK, int NTH, bool DIRECT> struct Operand {
  static constexpr int NP = Frag<T>::NP, E = 16 / (int)sizeof(T);
  static_assert(!DIRECT || NP == 1, "fp32 is split on its way to LDS");
  static constexpr int LINES = LAY == LAY_K ? ROWS : BK, WIDTH = LAY == LAY_K ? BK : ROWS;
  static constexpr int PITCH = WIDTH * 2 + (DIRECT ? 0 : LAY == LAY_K ? 16 : 64);
  static constexpr int PLANE = LINES * PITCH, BYTES = PLANE * NP;
  static constexpr int UPL = WIDTH / E, UNITS = LINES * UPL, U = (UNITS + NTH - 1) / NTH;
  static_assert(!DIRECT || (UNITS % NTH == 0 && (LAY == LAY_R || UPL == 4 || UPL == 8)), "whole waves, known line widths");
  u32x4 r[DIRECT ? 1 : U];
  const T* p[U];          // this thread's units of the next step
  int left[U];            // LAY_R: columns from the unit to the matrix's edge
  bool edge;              // LAY_R: the tile has units that are cut by the edge

  // which 16-byte piece of line `line` lies at piece `at`
  static __device__ __forceinline__ int piece(int line, int at) {
    if constexpr (!DIRECT) return at;
    else if constexpr (LAY == LAY_K) return at ^ ((line >> (UPL == 8 ? 1 : 2)) & (UPL - 1));   // 16 neighbouring lines cover the banks
    else return at ^ ((line & 3) << 1 & (UPL - 1));
  }
  __device__ __forceinline__ void init(const void* base, int64_t ld, int64_t row0, int64_t rows, int64_t r0, int tid) {
    edge = LAY == LAY_R && rows % E != 0 && row0 + WIDTH > rows;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = tid + NTH * i, line = u / UPL, c = piece(line, u % UPL) * E;
      if constexpr (LAY == LAY_K) {
        p[i] = static_cast<const T*>(base) + min(row0 + line, rows - 1) * ld + r0 + c;
      } else {
        const bool in = row0 + c < rows;
        p[i] = static_cast<const T*>(base) + (r0 + line) * ld + (in ? row0 + c : 0);
        left[i] = (int)min<int64_t>(E, in ? rows - row0 - c : rows);
      }
    }
  }
  // the unit of a step that is not whole
  __device__ __forceinline__ u32x4 cut(int i, int64_t left_r, int tid) const {
    const int u = tid + NTH * i, line = u / UPL;
    if constexpr (LAY == LAY_K) return load_unit(p[i], left_r - piece(line, u % UPL) * E);
    else return load_unit(p[i], line < left_r ? left[i] : 0);
  }
  // A whole step.  wave0: the first thread of this wave, as a scalar.
  __device__ __forceinline__ void load(int64_t ld, char* tile, int wave0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if constexpr (DIRECT) {
        // As asm without outputs: for the builtin the compiler waits for every such load before the next read of LDS, which would
        // undo the prefetch; here the barrier of the main loop counts them (its own waits only become stricter by them).  The
        // hardware writes lane l's 16 bytes at m0 + 16 l.
        const unsigned at = (unsigned)(uintptr_t)(tile + (i * NTH + wave0) * 16);   // the low half of an LDS address is its offset
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p[i]), "s"(at) : "memory", "m0");
      } else __builtin_memcpy(&r[i], p[i], 16);
      p[i] += LAY == LAY_K ? BK : BK * ld;
    }
  }
  // Any other step: left_r reduction indices from its first to the end.
  __device__ __forceinline__ void load_cut(int64_t ld, int64_t left_r, char* tile, int tid) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const u32x4 w = cut(i, left_r, tid);
      if constexpr (DIRECT) *reinterpret_cast<u32x4*>(tile + (i * NTH + tid) * 16) = w;
      else r[i] = w;
      p[i] += LAY == LAY_K ? BK : BK * ld;
    }
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int u = tid + NTH * i;
        if (UNITS % NTH == 0 || u < UNITS) {
          char* q = tile + (u / UPL) * PITCH + (u % UPL) * E * 2;
          if constexpr (NP == 1) *reinterpret_cast<u32x4*>(q) = r[i];
          else {
            u32x2 h, m, l;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x0 = __uint_as_float(r[i][2 * e]), x1 = __uint_as_float(r[i][2 * e + 1]);
              h[e] = pack_bf16(x0, x1);
              const float a0 = x0 - half_lo(h[e]), a1 = x1 - half_hi(h[e]);
              m[e] = pack_bf16(a0, a1);
              l[e] = pack_bf16(a0 - half_lo(m[e]), a1 - half_hi(m[e]));
            }
            *reinterpret_cast<u32x2*>(q) = h;
            *reinterpret_cast<u32x2*>(q + PLANE) = m;
            *reinterpret_cast<u32x2*>(q + 2 * PLANE) = l;
          }
        }
      }
    }
  }
  // rows row .. row + 31 (one a lane), reduction indices 16 ks + 8 (lane / 32) + 0..7
  static __device__ __forceinline__ typename Frag<T>::F frag(const char* tile, int plane, int row, int ks, int lane) {
    const char* t = tile + plane * PLANE;
    if constexpr (LAY == LAY_K) {
      const int line = row + (lane & 31);
      return __builtin_bit_cast(typename Frag<T>::F, *reinterpret_cast<const u32x4*>(t + line * PITCH + piece(line, 2 * ks + (lane >> 5)) * 16));
    } else {
      // a 16-lane group names four lines of 16 columns, 8 bytes a lane, and every lane gets its column of them
      typedef s16x4 __attribute__((address_space(3))) * lds_p;
      const int line = 16 * ks + 8 * (lane >> 5) + ((lane >> 2) & 3), col = row + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const char* a = t + line * PITCH + piece(line, col >> 3) * 16 + (col & 7) * 2;   // line + 4 has the same permutation
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + 4 * PITCH));
      return __builtin_bit_cast(typename Frag<T>::F, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

template <typename T, int N> __device__ __forceinline__ void load_row(const T* p, int left, float (&x)[N]) {
  if (left >= N) {
    T v[N];
    __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = e < left ? (float)p[e] : 0.0f;
  }
}
template <typename T, int N> __device__ __forceinline__ void store_row(T* p, int left, const float (&x)[N]) {
  if (left >= N) {
    T v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (T)x[e];
    __builtin_memcpy(p, v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) p[e] = (T)x[e];
  }
}

// An activation's slope (magnitude below 1.25) in 16 bits beside 16-bit types: its sign and the fourth root of its magnitude in 15 bits,
// steps of 1/30720.  What the backward pass needs of z, in z's room: rounded z, or slopes in the type itself, would add as much error to
// the gradients as their own rounding.  Steps of a root get finer with the slope, so that saturated units keep theirs: off by 2^-13.9
// of a slope of 1, 2^-12.9 at 2^-4, 2^-10.4 at 2^-14, 2^-9.9 at 2^-16 (fp16 itself: 2^-11 down to 2^-14, 2^-9 at 2^-16), and zero only
// below 2^-63.  Zero and one are exact, the two square roots and the decoding add 2^-20.  All ones stand for NaN.
struct Slope16 {
  static constexpr float STEPS = 30720.0f, BACK = 1.0f / (STEPS * STEPS * STEPS * STEPS);
  static __device__ __forceinline__ unsigned pack(float s) {
    const float a = __builtin_fabsf(s), q = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(a));
    const unsigned u = (unsigned)(int)__builtin_fmaf(q, STEPS, 0.5f);
    return (a < 1.25f ? u : 0x7fffu) | ((__float_as_uint(s) >> 16) & 0x8000u);
  }
  static __device__ __forceinline__ float unpack(unsigned u) {
    const float q = (float)(int)(u & 0x7fffu), q2 = q * q, a = q2 * q2 * BACK;
    return (u & 0x7fffu) == 0x7fffu ? __builtin_nanf("") : (u & 0x8000u) ? -a : a;
  }
};
template <typename T> struct SlopeOf { typedef unsigned short S; };
template <> struct SlopeOf<float> { typedef float S; };
template <typename S> __device__ __forceinline__ void load_slopes(const S* p, int left, float (&x)[8]) {
  if constexpr (sizeof(S) == 4) load_row<float, 8>(p, left, x);
  else {
    const u32x4 w = load_unit<__bf16>(reinterpret_cast<const __bf16*>(p), left);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Slope16::unpack((w[e / 2] >> (16 * (e & 1))) & 0xffffu);
  }
}
template <typename S> __device__ __forceinline__ void store_slopes(S* p, int left, const float (&x)[8]) {
  if constexpr (sizeof(S) == 4) store_row<float, 8>(p, left, x);
  else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = Slope16::pack(x[2 * e]) | Slope16::pack(x[2 * e + 1]) << 16;
    typedef u32x4 __attribute__((aligned(2))) unit;
    if (left >= 8) __builtin_nontemporal_store(w, reinterpret_cast<unit*>(p));
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) p[e] = (S)(w[e / 2] >> (16 * (e & 1)));
    }
  }
}

// Consecutive blocks go to the 8 XCDs in turn: each XCD gets a run of neighbouring tiles, so that its L2 holds what they share.
struct Tile { int split, n0; int64_t m0, r0, r1; bool none; };
template <int BM, int BN> __device__ __forceinline__ Tile tile_of(const MmP& p) {
  Tile t;
  const int tiles = p.m_tiles * p.n_tiles, per = gridDim.x / 8;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3), tile = id % tiles;
  t.none = id >= p.blocks;                                // the grid is padded to a multiple of 8
  t.split = id / tiles;
  t.m0 = (int64_t)(tile / p.n_tiles) * BM;
  t.n0 = (tile % p.n_tiles) * BN;
  t.r0 = t.split * p.r_split;
  t.r1 = min(p.R, t.r0 + p.r_split);
  return t;
}

// Eight values in units that are not read again soon: past the L2, which holds what the tiles share (W and the rows of x)
template <typename T> __device__ __forceinline__ void stream8(T* p, const T (&x)[8]) {
  typedef u32x4 __attribute__((aligned(2))) unit;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    u32x4 w;
    __builtin_memcpy(&w, x + i * 16 / sizeof(T), 16);
    __builtin_nontemporal_store(w, reinterpret_cast<unit*>(p) + i);
  }
}
template <typename T> __device__ __forceinline__ void stream_row(T* p, int left, const float (&x)[8]) {
  if (left >= 8) {
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)x[e];
    stream8(p, v);
  } else store_row<T, 8>(p, left, x);
}

template <typename T, int ACT, bool RES> __device__ __forceinline__ void finish8(const MmP& p, int64_t at, int left, float (&v)[8], const float (&bias)[8], const T (&res)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += bias[e];
  if (ACT != MRL_ACT_NONE && p.slope) {
    typedef typename SlopeOf<T>::S S;
    float d[8];
    act_slope<8>(ACT, v, d);
    store_slopes(static_cast<S*>(p.slope) + at, left, d);
  }
  act_fwd<8>(ACT, v);
  if constexpr (RES) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += (float)res[e];
  }
  stream_row<T>(static_cast<T*>(p.y) + at, left, v);
}

// The epilogue of a wave's TM x TN accumulators, by itself: 32 rows at a time go through its own piece of LDS and leave in units of 8
// columns, whole cache lines of a row.  The residuals (RES: there are any; without, the kernel is smaller by their registers) are on
// their way since the last step.
template <typename T, int TM, int TN, bool PLAIN, bool RES> struct WaveEpilogue {
  static constexpr int W = TN * 32, EP = W + 4, BYTES = 32 * EP * 4, UPR = W / 8, UNITS = 32 * UPR / 64;
  typedef T row8[8];
  static constexpr int AHEAD = TM < 2 || sizeof(T) == 4 ? 1 : 2;   // 32-row pieces of the residual in registers
  typedef row8 Residual[AHEAD][UNITS];
  static __device__ __forceinline__ void fetch(const MmP& p, int64_t m, int n, int lane, row8 (&res)[UNITS]) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int u = lane + 64 * i, c = n + (u % UPR) * 8, left = p.N - c;
      const int64_t row = m + u / UPR;
      if (row < p.M && left > 0) {
        const T* q = static_cast<const T*>(p.residual) + row * p.N + c;
        if (left >= 8) {
          typedef u32x4 __attribute__((aligned(2))) unit;
#pragma unroll
          for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const unit*>(q) + h);
            __builtin_memcpy(res[i] + h * 16 / sizeof(T), &w, 16);
          }
        }
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) res[i][e] = e < left ? q[e] : (T)0.0f;
        }
      }
    }
  }
  // the first pieces of the residual: issued before the wave's last products
  static __device__ __forceinline__ void fetch_first(const MmP& p, int64_t m, int n, int lane, Residual& res) {
    if (!RES) return;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(p, m + 32 * i, n, lane, res[i]);
  }
  template <int ACT>
  static __device__ __forceinline__ void run_act(const MmP& p, const Tile& t, float* lds, const f32x16 (&acc)[TN][TM], int64_t m, int n, int lane, Residual& res) {
    float bias[8];
    const int c = n + (lane % UPR) * 8, left = p.N - c;     // 64 is a multiple of UPR: a lane's columns stay
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = 0.0f;
    if (!PLAIN && p.bias && left > 0) load_row<T, 8>(static_cast<const T*>(p.bias) + c, left, bias);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(lds + (lane & 31) * EP + j * 32 + 8 * q + 4 * (lane >> 5)) =
              f32x4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
      __builtin_amdgcn_wave_barrier();                      // one wave: its LDS operations stay in order
#pragma unroll
      for (int k = 0; k < UNITS; ++k) {
        const int u = lane + 64 * k;
        const int64_t row = m + 32 * i + u / UPR;
        float v[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 s = *reinterpret_cast<const f32x4*>(lds + (u / UPR) * EP + (u % UPR) * 8 + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * h + e] = s[e];
        }
        if (row < p.M && left > 0) {
          const int64_t at = row * p.N + c;
          if constexpr (PLAIN && std::is_same_v<T, _Float16>) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= p.gain;
          }
          if (PLAIN && p.slab) store_row<float, 8>(p.slab + (int64_t)t.split * p.M * p.N + at, left, v);
          else if (PLAIN) store_row<T, 8>(static_cast<T*>(p.y) + at, left, v);
          else finish8<T, ACT, RES>(p, at, left, v, bias, res[i % AHEAD][k]);
        }
      }
      if (RES && i + AHEAD < TM) fetch(p, m + 32 * (i + AHEAD), n, lane, res[i % AHEAD]);
      __builtin_amdgcn_wave_barrier();
    }
  }
  static __device__ __forceinline__ void run(const MmP& p, const Tile& t, float* lds, const f32x16 (&acc)[TN][TM], int64_t m, int n, int lane, Residual& res) {
    if constexpr (PLAIN) run_act<MRL_ACT_NONE>(p, t, lds, acc, m, n, lane, res);
    else switch (p.act) {                                   // one straight path per activation
      case MRL_ACT_SILU: run_act<MRL_ACT_SILU>(p, t, lds, acc, m, n, lane, res); break;
      case MRL_ACT_ELU: run_act<MRL_ACT_ELU>(p, t, lds, acc, m, n, lane, res); break;
      case MRL_ACT_RELU: run_act<MRL_ACT_RELU>(p, t, lds, acc, m, n, lane, res); break;
      case MRL_ACT_TANH: run_act<MRL_ACT_TANH>(p, t, lds, acc, m, n, lane, res); break;
      case MRL_ACT_GELU: run_act<MRL_ACT_GELU>(p, t, lds, acc, m, n, lane, res); break;
      default: run_act<MRL_ACT_NONE>(p, t, lds, acc, m, n, lane, res); break;
    }
  }
};

// WM x WN waves over the tile, WK waves over the reduction inside a step; NST stages in LDS, NST - 1 steps of loads in flight (DIRECT),
// or loads through registers one step ahead with NST 1 or 2 stages.
template <typename T, int BM, int BN, int BK, int WM, int WN, int WK, int LA, int LB, int NST, bool DIRECT, bool RES>
__global__ __launch_bounds__(WM * WN * WK * 64, DIRECT && NST == 3 ? 3 : 2) void mm_kernel(const MmP p) {
  constexpr int NTH = WM * WN * WK * 64, TM = BM / WM / 32, TN = BN / WN / 32, KS = BK / 16 / WK, NP = Frag<T>::NP;
  constexpr bool PLAIN = LB == LAY_R;                      // a gradient: no epilogue but the store
  typedef Operand<T, LA, BM, BK, NTH, DIRECT> OA;
  typedef Operand<T, LB, BN, BK, NTH, DIRECT> OB;
  typedef typename Frag<T>::F F;
  typedef WaveEpilogue<T, TM, TN, PLAIN, RES> WE;
  static_assert(WK == 1 || (TM == 1 && TN == 1), "shared reductions: one tile a wave");
  constexpr int STAGE = OA::BYTES + OB::BYTES, EBYTES = WE::BYTES * WM * WN * WK;
  constexpr int LDS = NST * STAGE > EBYTES ? NST * STAGE : EBYTES;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  const Tile t = tile_of<BM, BN>(p);
  if (t.none) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wk = wave % WK, wn = wave / WK % WN, wm = wave / (WK * WN);

  OA oa;
  OB ob;
  oa.init(p.a, p.lda, t.m0, p.M, t.r0, tid);
  ob.init(p.b, p.ldb, t.n0, p.N, t.r0, tid);
  f32x16 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.0f;

  const int steps = (int)((t.r1 - t.r0 + BK - 1) / BK);
  auto multiply = [&](const char* st) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int ks = wk * KS + k;
      F a[NP][TM], b[NP][TN];
#pragma unroll
      for (int q = 0; q < NP; ++q) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a[q][i] = OA::frag(st, q, (wm * TM + i) * 32, ks, lane);
#pragma unroll
        for (int j = 0; j < TN; ++j) b[q][j] = OB::frag(st + OA::BYTES, q, (wn * TN + j) * 32, ks, lane);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if constexpr (NP == 3) {
            acc[j][i] = Frag<T>::mul(b[2][j], a[0][i], acc[j][i]);
            acc[j][i] = Frag<T>::mul(b[0][j], a[2][i], acc[j][i]);
            acc[j][i] = Frag<T>::mul(b[1][j], a[1][i], acc[j][i]);
            acc[j][i] = Frag<T>::mul(b[1][j], a[0][i], acc[j][i]);
            acc[j][i] = Frag<T>::mul(b[0][j], a[1][i], acc[j][i]);
          }
          acc[j][i] = Frag<T>::mul(b[0][j], a[0][i], acc[j][i]);
        }
    }
  };
  // Steps that are loaded without checks: those of BK indices; beside a cut edge, whose units reach up to 7 elements, so at most as
  // many lines, too far, only those that far from the matrix's end.
  const int64_t span = t.r1 - t.r0, room = oa.edge || ob.edge ? min(span, p.R - t.r0 - 8) : span;
  const int whole = (int)(room > 0 ? room / BK : 0), wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);
  auto load = [&](int s, char* st) {
    if (s < whole) {
      oa.load(p.lda, st, wave0);
      ob.load(p.ldb, st + OA::BYTES, wave0);
    } else {
      oa.load_cut(p.lda, span - (int64_t)s * BK, st, tid);
      ob.load_cut(p.ldb, span - (int64_t)s * BK, st + OA::BYTES, tid);
    }
  };
  const int64_t wave_m = t.m0 + wm * TM * 32;
  const int wave_n = t.n0 + wn * TN * 32;
  typename WE::Residual res;
  auto store = [&](char* st) {
    oa.store(st, tid);
    ob.store(st + OA::BYTES, tid);
  };
  if constexpr (DIRECT) {
    constexpr int L = OA::U + OB::U;                       // loads of a step, each counted once by vmcnt
    static_assert((NST - 2) * L < 64, "vmcnt");
#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
      if (s < steps) load(s, lds + s * STAGE);
    int at = 0;
    for (int s = 0; s < steps; ++s) {
      // This wave's share of stage s has landed when no more than the later steps' loads are outstanding; the last steps, which
      // have fewer behind them (and maybe a cut one, loaded through registers), wait for everything.  Behind the barrier every
      // wave's share has landed and every wave has left the stage that is filled next.  (__syncthreads would wait for all loads.)
      if (s + NST - 1 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NST - 2) * L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (s + NST - 1 < steps) load(s + NST - 1, lds + (at == 0 ? NST - 1 : at - 1) * STAGE);
      if (s + 1 == steps) WE::fetch_first(p, wave_m, wave_n, lane, res);
      multiply(lds + at * STAGE);
      at = at + 1 == NST ? 0 : at + 1;
    }
  } else if constexpr (NST == 2) {
    if (steps > 0) {
      load(0, lds);
      store(lds);
    }
    for (int s = 0; s < steps; ++s) {
      if (s + 1 < steps) load(s + 1, lds);
      else WE::fetch_first(p, wave_m, wave_n, lane, res);
      __syncthreads();                                     // stage s is written, and every wave has left the one that s + 1 goes to
      multiply(lds + (s & 1) * STAGE);
      if (s + 1 < steps) store(lds + ((s + 1) & 1) * STAGE);
    }
  } else {
    if (steps > 0) load(0, lds);
    for (int s = 0; s < steps; ++s) {
      store(lds);
      if (s + 1 < steps) load(s + 1, lds);
      else WE::fetch_first(p, wave_m, wave_n, lane, res);
      __syncthreads();
      multiply(lds);
      __syncthreads();
    }
  }
  if (steps == 0) WE::fetch_first(p, wave_m, wave_n, lane, res);
  __syncthreads();                                         // the stages are free
  float* ep = reinterpret_cast<float*>(lds) + wave * (WE::BYTES / 4);
  if constexpr (WK > 1) {                                  // the waves' shares, added in order by the first
    if (wk > 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) ep[e * 64 + lane] = acc[0][0][e];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int k = 1; k < WK; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[0][0][e] += ep[k * (WE::BYTES / 4) + e * 64 + lane];
  }
  WE::run(p, t, ep, acc, wave_m, wave_n, lane, res);
}

// dz = dy slope, rounded to T as an operand of the two products (with the results' own rounding that makes 1.4 times the error of one;
// a second term would double both products: 180 us of 400 at 32768 x 512 -> 2048), and the sums of its columns, unrounded, over this block's
// rows -> part [blocks in y][N], or db where one block has all rows (a launch less for small batches).  32 units of 8 columns x 8 rows a block.
// fp16 beside SiLU and GELU, whose slopes pass one, keeps shrink dz = dz / 2, which has room for every finite dy, and the products are doubled
// (exactly, in fp32): dz itself would be infinite from dy = 58000 on.  Subnormal values of dz lose one more bit by it.
// cuts: a slope of zero drops dy, whatever it is (the rectifier, as in torch); beside the other activations a dy that is not finite stays so.
template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const typename SlopeOf<T>::S* __restrict__ slope, const T* __restrict__ dy, T* __restrict__ dz, float* __restrict__ part,
                                                 T* __restrict__ db, int64_t M, int N, int rows, bool cuts, float shrink) {
  __shared__ float red[8][32 * 8 + 1];
  const int cu = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + cu) * 8, left = N - c;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.0f;
  if (left > 0) {
    const int64_t m1 = min(M, ((int64_t)blockIdx.y + 1) * rows);
    constexpr int U = sizeof(T) == 2 ? 4 : 2;               // rows in flight
    for (int64_t m = (int64_t)blockIdx.y * rows + rl; m < m1; m += 8 * U) {
      float d[U][8], g[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (m + 8 * u < m1) {
          load_row<T, 8>(dy + (m + 8 * u) * N + c, left, d[u]);
          if (slope) load_slopes(slope + (m + 8 * u) * N + c, left, g[u]);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (m + 8 * u < m1) {
          if (slope) {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[u][e] = cuts && g[u][e] == 0.0f ? 0.0f : d[u][e] * g[u][e];
            if constexpr (std::is_same_v<T, _Float16>) {
              float half[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) half[e] = d[u][e] * shrink;
              store_row<T, 8>(dz + (m + 8 * u) * N + c, left, half);
            } else store_row<T, 8>(dz + (m + 8 * u) * N + c, left, d[u]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] += d[u][e];
        }
    }
  }
  if (!part && !db) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[rl][cu * 8 + e] = s[e];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col < N) {
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) a += red[k][threadIdx.x];
    if (db) db[col] = (T)a;
    else part[(int64_t)blockIdx.y * N + col] = a;
  }
}

// out[c] = sum over rows of part [rows][n]: 32 columns a block, 32 threads a column
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ part, int64_t rows, int n, T* __restrict__ out) {
  __shared__ float red[32][33];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float a = 0.0f;
  if (c < n) {
    constexpr int U = 8;
    for (int64_t r = rl; r < rows; r += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = r + 32 * u < rows ? part[(r + 32 * u) * n + c] : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) a += v[u];
    }
  }
  red[rl][cl] = a;
  __syncthreads();
  if (rl == 0 && c < n) {
    float s = 0.0f;
    for (int k = 0; k < 32; ++k) s += red[k][cl];
    out[c] = (T)s;
  }
}

// dW = sum of the splits' slabs, four values a thread
template <typename T>
__global__ __launch_bounds__(256) void slab_sum_kernel(const float* __restrict__ slab, int splits, int64_t n, T* __restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int left = (int)min<int64_t>(4, n - i);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;                                      // slabs in flight
  for (int k = 0; k < splits; k += U) {
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < splits) load_row<float, 4>(slab + (k + u) * n + i, left, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < splits) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[u][e];
      }
  }
  store_row<T, 4>(out + i, left, s);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
int check(const mrl_linear* p, const char* what) {
  if (!p) MEM_FAIL(MRL_EINVAL, "%s: null description", what);
  if (p->dtype < MRL_F32 || p->dtype > MRL_F16) MEM_FAIL(MRL_EINVAL, "%s: dtype %d (float32, bfloat16 or float16)", what, p->dtype);
  if (p->act < MRL_ACT_NONE || p->act > MRL_ACT_GELU) MEM_FAIL(MRL_EINVAL, "%s: activation %d", what, p->act);
  if (p->rows < 0 || p->inputs < 0 || p->outputs < 0) MEM_FAIL(MRL_EINVAL, "%s: rows %lld, inputs %d, outputs %d", what, (long long)p->rows, p->inputs, p->outputs);
  if (p->rows > (int64_t(1) << 30) || p->inputs > (1 << 24) || p->outputs > (1 << 24)) MEM_FAIL(MRL_EINVAL, "%s: sizes beyond 2^30 rows or 2^24 columns", what);
  if (p->rows > 1 && p->x_stride < p->inputs) MEM_FAIL(MRL_EINVAL, "%s: x_stride %lld below %d inputs", what, (long long)p->x_stride, p->inputs);
  // tiles of at least 128 x 128 where there are many, 256 threads each, and a grid has less than 2^32 of them
  if (cdiv(std::max<int64_t>(p->rows, p->inputs), 128) * cdiv(std::max(p->inputs, p->outputs), 128) >= (int64_t(1) << 23)) MEM_FAIL(MRL_EINVAL, "%s: %lld rows, %d inputs, %d outputs: over 2^23 tiles", what, (long long)p->rows, p->inputs, p->outputs);
  return MRL_OK;
}

// Tile edge: the largest whose tiles fill the card; at 32 the block's waves share the reduction.  Measured, at the rule's edge and at
// its neighbours: dx of 32768 x 2048 -> 512, bf16: 256: 70 us, 128: 82, 64: 113.  Forward 4099 x 333 -> 777, fp16: 64: 18 us, 128: 21,
// 32: 25.  64 x 512 -> 512, bf16: 32: 4.9 us, 64: 5.8.  fp32 32768 x 256 -> 512: 256 (128 x 256): 63 us, 128: 66, 64: 72.
int edge_of(int64_t m, int64_t n, int dtype) {
  if (cdiv(m, dtype == MRL_F32 ? 128 : 256) * cdiv(n, 256) >= 200 && n >= 192) return 256;
  if (cdiv(m, 128) * cdiv(n, 128) >= 256) return 128;
  if (cdiv(m, 64) * cdiv(n, 64) >= 256) return 64;
  return 32;
}

// rows on 16-byte addresses, for the loads that write LDS themselves
bool direct_ok(const void* base, int64_t ld, int es) { return ((uintptr_t)base & 15) == 0 && ld * es % 16 == 0; }

template <typename T, int LA, int LB, bool RES> void multiply_as(MmP& a, int edge, int splits, hipStream_t st) {
  const bool direct = sizeof(T) == 2 && direct_ok(a.a, a.lda, 2) && direct_ok(a.b, a.ldb, 2);
  const bool wide = sizeof(T) == 4 && edge == 256;          // fp32: 128 x 256
  // 256 x 256 forward: not beside a residual, for which its accumulators leave no registers.  SiLU, bf16: 16384 x 2048 -> 2048 144 us,
  // 128: 177; 32768 x 512 -> 2048 97 and 107, with its slope 134 and 143; 32768 x 256 -> 1024 39 and 43.
  // 128 x 128 forward: three stages, so that three blocks share a CU and one's epilogue runs beside the others' products: 32768 x 512 ->
  // 2048 with SiLU, slope and residual 160 us, with two blocks and three or four stages 173 to 175.  Gradients have a
  // short epilogue and keep four stages (109 us, three: 113).
  const bool lean = LB == LAY_R || (!RES && a.R >= 256);
  if (edge == 256 && !wide && !(direct && lean)) edge = 128;
  a.m_tiles = (int)cdiv(a.M, wide ? 128 : edge);
  a.n_tiles = (int)cdiv(a.N, edge);
  a.blocks = a.m_tiles * a.n_tiles * splits;
  const dim3 grid((unsigned)(cdiv(a.blocks, 8) * 8));
  if constexpr (sizeof(T) == 4) {
    if (wide) hipLaunchKernelGGL((mm_kernel<T, 128, 256, 32, 2, 4, 1, LA, LB, 1, false, RES>), grid, dim3(512), 0, st, a);
    else if (edge == 128) hipLaunchKernelGGL((mm_kernel<T, 128, 128, 32, 2, 2, 1, LA, LB, 1, false, RES>), grid, dim3(256), 0, st, a);
    else if (edge == 64) hipLaunchKernelGGL((mm_kernel<T, 64, 64, 32, 2, 2, 1, LA, LB, 1, false, RES>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mm_kernel<T, 32, 32, 64, 1, 1, 4, LA, LB, 1, false, RES>), grid, dim3(256), 0, st, a);
  } else if (direct) {
    if constexpr (!RES) {
      if (edge == 256) {
        hipLaunchKernelGGL((mm_kernel<T, 256, 256, 32, 2, 4, 1, LA, LB, 4, true, false>), grid, dim3(512), 0, st, a);
        return;
      }
    }
    if (edge == 128) hipLaunchKernelGGL((mm_kernel<T, 128, 128, 32, 2, 2, 1, LA, LB, LB == LAY_K ? 3 : 4, true, RES>), grid, dim3(256), 0, st, a);
    else if (edge == 64) hipLaunchKernelGGL((mm_kernel<T, 64, 64, 64, 2, 2, 1, LA, LB, 4, true, RES>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mm_kernel<T, 32, 32, 64, 1, 1, 4, LA, LB, 8, true, RES>), grid, dim3(256), 0, st, a);
  } else {
    if (edge == 128) hipLaunchKernelGGL((mm_kernel<T, 128, 128, 64, 2, 2, 1, LA, LB, 2, false, RES>), grid, dim3(256), 0, st, a);
    else if (edge == 64) hipLaunchKernelGGL((mm_kernel<T, 64, 64, 64, 2, 2, 1, LA, LB, 2, false, RES>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mm_kernel<T, 32, 32, 64, 1, 1, 4, LA, LB, 2, false, RES>), grid, dim3(256), 0, st, a);
  }
}

template <typename T, int LA, int LB> void multiply(MmP& a, int edge, int splits, hipStream_t st) {
  if constexpr (LB == LAY_K) {
    if (a.residual) return multiply_as<T, LA, LB, true>(a, edge, splits, st);
  }
  multiply_as<T, LA, LB, false>(a, edge, splits, st);
}

struct Plan { int edge_x, edge_w, splits; int64_t r_split; int rows, parts; int64_t dz, part, slab, total; };

Plan plan_of(const mrl_linear* p) {
  Plan r{};
  const int64_t es = p->dtype == MRL_F32 ? 4 : 2;
  r.edge_x = edge_of(p->rows, p->inputs, p->dtype);
  // dW: the largest edge of which there are 64 tiles (128 at 256), the rows split until 512 blocks (256 of the large ones) run, each
  // with at least 1024 rows (512 at 128): more splits cost more in their sums than they win.  8192 x 8192 over 8192 rows, bf16: 256:
  // 1.01 ms, 128: 1.39.  2048 x 512 over 32768: 128: 82 us, 256: 92, 64: 104.  512 x 512 over 4096: 64: 12 us, 128: 20.
  auto tiles_of = [&](int edge) { return std::max<int64_t>(1, cdiv(p->outputs, edge) * cdiv(p->inputs, edge)); };
  r.edge_w = p->dtype != MRL_F32 && tiles_of(256) >= 128 ? 256 : tiles_of(128) >= 64 ? 128 : std::min(p->inputs, p->outputs) >= 48 ? 64 : 32;
  const int64_t tiles = tiles_of(r.edge_w);
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>(cdiv(r.edge_w == 256 ? 256 : 512, tiles), p->rows / (r.edge_w >= 128 ? 512 : 1024)));
  r.r_split = std::max<int64_t>(64, cdiv(cdiv(p->rows, splits), 64) * 64);
  r.splits = (int)std::max<int64_t>(1, cdiv(p->rows, r.r_split));
  // dz: blocks of 256 columns, about 2048 of them; one alone where it has all rows in flight at once
  const int64_t cols = std::max<int64_t>(1, cdiv(p->outputs, 256));
  r.rows = p->rows <= 32 ? 32 : (int)std::max<int64_t>(8, cdiv(cdiv(p->rows * cols, 2048), 8) * 8);
  r.parts = (int)std::max<int64_t>(1, cdiv(p->rows, r.rows));
  auto up = [](int64_t n) { return cdiv(n, 256) * 256; };
  r.dz = p->act == MRL_ACT_NONE ? 0 : up(p->rows * p->outputs * es);
  r.part = up((int64_t)r.parts * p->outputs * 4);
  r.slab = r.splits > 1 ? up((int64_t)r.splits * p->outputs * p->inputs * 4) : 0;
  r.total = r.dz + r.part + r.slab;
  return r;
}

template <typename T>
int forward(const mrl_linear* p, const void* x, const void* w, const void* bias, const void* residual, void* y, void* slope, hipStream_t st) {
  MmP a{};
  a.a = x; a.lda = p->x_stride; a.b = w; a.ldb = p->inputs; a.M = (int)p->rows; a.N = p->outputs; a.R = p->inputs; a.r_split = std::max(p->inputs, 1);
  a.y = y; a.bias = bias; a.residual = residual; a.slope = slope; a.act = p->act;
  multiply<T, LAY_K, LAY_K>(a, edge_of(p->rows, p->outputs, p->dtype), 1, st);
  return MRL_OK;
}

template <typename T>
int backward(const mrl_linear* p, const void* x, const void* w, const void* slope, const void* dy, void* dx, void* dw, void* db, char* ws, hipStream_t st) {
  const Plan r = plan_of(p);
  T* dz = reinterpret_cast<T*>(ws);
  float* part = reinterpret_cast<float*>(ws + r.dz);
  float* slab = reinterpret_cast<float*>(ws + r.dz + r.part);
  const bool act = p->act != MRL_ACT_NONE, whole = p->rows > 0 && r.parts == 1;
  const bool halves = p->dtype == MRL_F16 && (p->act == MRL_ACT_SILU || p->act == MRL_ACT_GELU);
  if (p->rows > 0 && (db || (act && (dx || dw))))
    hipLaunchKernelGGL((dz_kernel<T>), dim3((unsigned)cdiv(p->outputs, 256), r.parts), dim3(256), 0, st,
                       act ? static_cast<const typename SlopeOf<T>::S*>(slope) : nullptr, static_cast<const T*>(dy), dz, db && !whole ? part : nullptr,
                       whole ? static_cast<T*>(db) : nullptr, p->rows, p->outputs, r.rows, p->act == MRL_ACT_RELU, halves ? 0.5f : 1.0f);
  if (db && !whole) hipLaunchKernelGGL((column_sum_kernel<T>), dim3((unsigned)cdiv(p->outputs, 32)), dim3(1024), 0, st, part, p->rows > 0 ? r.parts : 0, p->outputs, static_cast<T*>(db));
  const void* d = act ? static_cast<const void*>(dz) : dy;
  if (dx && p->rows > 0 && p->inputs > 0) {
    MmP a{};
    a.gain = halves ? 2.0f : 1.0f; a.a = d; a.lda = p->outputs; a.b = w; a.ldb = p->inputs; a.M = (int)p->rows; a.N = p->inputs; a.R = p->outputs; a.r_split = p->outputs; a.y = dx;
    multiply<T, LAY_K, LAY_R>(a, r.edge_x, 1, st);
  }
  if (dw && p->inputs > 0) {
    MmP a{};
    a.gain = halves ? 2.0f : 1.0f; a.a = d; a.lda = p->outputs; a.b = x; a.ldb = p->x_stride; a.M = p->outputs; a.N = p->inputs; a.R = p->rows; a.r_split = r.r_split;
    if (r.splits > 1) a.slab = slab;
    else a.y = dw;
    multiply<T, LAY_R, LAY_R>(a, r.edge_w, r.splits, st);
    const int64_t n = (int64_t)p->outputs * p->inputs;
    if (r.splits > 1) hipLaunchKernelGGL((slab_sum_kernel<T>), dim3((unsigned)cdiv(n, 1024)), dim3(256), 0, st, slab, r.splits, n, static_cast<T*>(dw));
  }
  return MRL_OK;
}

}  // namespace

extern "C" int mrl_linear_act(const mrl_linear* p, const void* x, const void* weight, const void* bias, const void* residual, void* y, void* slope, void* stream) {
  const char* what = "mrl_linear_act";
  const int rc = check(p, what);
  if (rc) return rc;
  if (p->rows == 0 || p->outputs == 0) return MRL_OK;
  if (!y || (p->inputs > 0 && (!x || !weight))) MEM_FAIL(MRL_EINVAL, "%s: null data", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == MRL_F32) forward<float>(p, x, weight, bias, residual, y, slope, st);
  else if (p->dtype == MRL_BF16) forward<__bf16>(p, x, weight, bias, residual, y, slope, st);
  else forward<_Float16>(p, x, weight, bias, residual, y, slope, st);
  MEM_CHECK_LAUNCH(what);
  return MRL_OK;
}

extern "C" int64_t mrl_linear_act_backward_workspace_bytes(const mrl_linear* p) {
  const int rc = check(p, "mrl_linear_act_backward_workspace_bytes");
  if (rc) return rc;
  return plan_of(p).total;
}

extern "C" int mrl_linear_act_backward(const mrl_linear* p, const void* x, const void* weight, const void* slope, const void* dy, void* dx, void* d_weight, void* d_bias,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mrl_linear_act_backward";
  const int rc = check(p, what);
  if (rc) return rc;
  if (p->outputs == 0) MEM_FAIL(MRL_EINVAL, "%s: no outputs", what);
  if (p->rows > 0) {
    if (!dy || (p->act != MRL_ACT_NONE && !slope)) MEM_FAIL(MRL_EINVAL, "%s: null dy or slope", what);
    if (p->inputs > 0 && ((dx && !weight) || (d_weight && !x))) MEM_FAIL(MRL_EINVAL, "%s: null x or weight", what);
  }
  const int64_t need = plan_of(p).total;
  if (need > 0 && (!workspace || workspace_bytes < need)) MEM_FAIL(MRL_ENOSPC, "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  if ((uintptr_t)workspace & 15) MEM_FAIL(MRL_EINVAL, "%s: workspace is not aligned", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  if (p->dtype == MRL_F32) backward<float>(p, x, weight, slope, dy, dx, d_weight, d_bias, ws, st);
  else if (p->dtype == MRL_BF16) backward<__bf16>(p, x, weight, slope, dy, dx, d_weight, d_bias, ws, st);
  else backward<_Float16>(p, x, weight, slope, dy, dx, d_weight, d_bias, ws, st);
  MEM_CHECK_LAUNCH(what);
  return MRL_OK;
}
