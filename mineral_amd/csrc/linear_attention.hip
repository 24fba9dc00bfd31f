// Linear attention with one decay per head for gfx950: whole sequences in chunks, their gradient, and single tokens.
//
//   S_t = lambda S_{t-1} + k_t v_t^T (S_{t-1} dropped where token t begins an episode),   o_t = S_t^T q_t
//
// A chunk of C tokens that starts with the state S needs three products and one update (i, j inside the chunk, same episode):
//   P_ij = lambda^(i-j) q_i.k_j (i >= j),   o_i = sum_j P_ij v_j + lambda^(i+1) S^T q_i,   S <- lambda^C S + sum_j lambda^(C-1-j) k_j v_j^T
// The gradients are the same scan with the operands in other places: dq = scan(do, v; k), and, backwards in time,
// dk = scan(v, do; q), dv = scan(k, q; do), whose state is the gradient of S (the last one's end is the initial state's gradient).
// Backwards the decay follows a token's write instead of preceding it (`off` 0 instead of 1).  One kernel serves all four.
//
// Layout: one block per (batch row, head, segment of the tokens), one wave for every 16 value columns, which holds all rows of its
// columns of S in MFMA accumulators for the whole segment.  The products are arranged so that every
// intermediate is the next product's operand where it lies: with 16x16x32 MFMAs a lane's accumulators of two stacked 16-row tiles
// are rows {4g..4g+3, 16+4g..16+4g+3} of its column (g = lane / 16), and any order of the reduction index serves as long as both
// operands share it, so S and P^T go from accumulators to operands without LDS; row-major operands lie in LDS in that order and are
// read in 16-byte pieces, token-major ones through the transposing LDS read, whose 16-lane groups return exactly four rows of
// a column.  Only q, k, v pass through LDS (registers hold the next chunk meanwhile).  The scores are computed by every wave:
// matrix work is not what bounds the kernel, an exchange through LDS with its barriers would.
//
// Precision: everything accumulates in fp32.  16-bit inputs multiply as they are (fp16 as two exact bf16 terms where the partner
// is an fp32 intermediate, whose range fp16 lacks); an fp32 intermediate enters a product as two bf16 terms (P, S: 2^-17 relative,
// below the rounding of the 16-bit outputs) or three (the weighted v of the state, which stays fp32: 2^-24).  fp32 inputs become
// three exact bf16 terms on their way to LDS and multiply in six products, like every intermediate beside them: 2^-23, and 2.7 times
// the rate of the fp32 MFMA.
//
// Bound: by memory where there are many sequences (8192 of 32 tokens, 64 x 64, fp32, states in and out: 111 us for 0.54 GB, 4.8 TB/s;
// their gradient about 275 us for 1.38 GB, 5.0 TB/s: its three scans run one after the other and read q, k, v and d_out again, 1.02 GB
// instead of 0.54); by the latency of one chunk after the other where few sequences are long: 4.5 us for 64 tokens in 16 bits at 64 x 64
// (272 blocks of 655 tokens: 49 us), 4.6 for 32 in fp32 (96 us), and 7 for 64 at 128 x 128, where each of eight waves computes all scores
// for its 16 columns and one block fills a CU (8 sequences of 16384 tokens, bf16: 27 us for the segments' states, 3.4 a chunk, 12 to join
// them, 57 for the outputs).
//
// Masked tokens: weights are applied by selection, and a chunk that holds an infinity or NaN is walked token by token (the same
// code with chunks of one), so that a zero weight never meets one: nothing of a later token or an earlier episode leaks.
#include "memory_common.hip.h"

using namespace mrl::mem;

namespace {

constexpr int MAX_ROLES = 3;

struct Role {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];   // batch, step (negative: backwards in time), head; elements
  void* out;
  int64_t os[3];
  const uint8_t* resets;         // of the first token in walking order, or null
  int64_t rs[2];                 // batch, step
  const float* s0;               // state on entry, element (row, col) at row * s_row + col * s_col; or null
  float* s1;                     // state at the end, or null
  int s_row, s_col;
  int dq, dv;                    // reduction width (q, k), output width (v)
  int off;                       // decays between the state on entry and the first token's reading
  float oscale, wscale;          // factor of the outputs; factor of every k v^T
  int vec;                       // all rows of q, k, v lie on 16-byte addresses
  int64_t ws;                    // this role's place in the workspace, floats
};

struct ScanP {
  Role role[MAX_ROLES];
  const float* log_decay;
  float* ws;
  int* flags;                    // [role][split][bh]: a reset inside that segment
  int T, seg, n_splits, H;
  int BH;
};

__device__ __forceinline__ double log2_decay(const float* log_decay, int h) { return (double)log_decay[h] * 1.4426950408889634; }
// decay ** n; n <= 0 gives 1, also for a decay of zero.  The exponent is formed in 64 bits, so a long distance loses nothing.
__device__ __forceinline__ float decay_pow(double l2, int n) {
  if (n <= 0) return 1.0f;
  const double x = l2 * n;
  if (x < -1000.0) return 0.0f;
  const double w = __builtin_rint(x);
  return __builtin_ldexpf(__builtin_amdgcn_exp2f((float)(x - w)), (int)fmin(w, 2000.0));
}

// ---- element types ----------------------------------------------------------------------------------------------------------
// Raw: a fragment as it comes from LDS; In: the same as operand next to an fp32 intermediate; De: an fp32 intermediate as operand of
// an output's product; Wt: as operand of the state's.
struct Planes1 { bf16x8 p[1]; };
struct Planes2 { bf16x8 p[2]; };
struct Planes3 { bf16x8 p[3]; };

__device__ __forceinline__ Planes2 split2(const f32x8 x) {
  Planes2 r;
  u32x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
    l[e] = pack_bf16(x[2 * e] - half_lo(h[e]), x[2 * e + 1] - half_hi(h[e]));
  }
  r.p[0] = __builtin_bit_cast(bf16x8, h);
  r.p[1] = __builtin_bit_cast(bf16x8, l);
  return r;
}
__device__ __forceinline__ Planes3 split3(const f32x8 x) {
  Planes3 r;
  u32x4 h, m, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
    const float a = x[2 * e] - half_lo(h[e]), b = x[2 * e + 1] - half_hi(h[e]);
    m[e] = pack_bf16(a, b);
    l[e] = pack_bf16(a - half_lo(m[e]), b - half_hi(m[e]));
  }
  r.p[0] = __builtin_bit_cast(bf16x8, h);
  r.p[1] = __builtin_bit_cast(bf16x8, m);
  r.p[2] = __builtin_bit_cast(bf16x8, l);
  return r;
}
__device__ __forceinline__ f32x4 mfma_bf(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ void mma(f32x4& c, const Planes1& a, const Planes2& b) {
  c = mfma_bf(a.p[0], b.p[1], c);
  c = mfma_bf(a.p[0], b.p[0], c);
}
__device__ __forceinline__ void mma(f32x4& c, const Planes2& a, const Planes1& b) {
  c = mfma_bf(a.p[1], b.p[0], c);
  c = mfma_bf(a.p[0], b.p[0], c);
}
__device__ __forceinline__ void mma(f32x4& c, const Planes2& a, const Planes2& b) {   // the product of both low terms is below 2^-16
  c = mfma_bf(a.p[1], b.p[0], c);
  c = mfma_bf(a.p[0], b.p[1], c);
  c = mfma_bf(a.p[0], b.p[0], c);
}
__device__ __forceinline__ void mma(f32x4& c, const Planes1& a, const Planes3& b) {
  c = mfma_bf(a.p[0], b.p[2], c);
  c = mfma_bf(a.p[0], b.p[1], c);
  c = mfma_bf(a.p[0], b.p[0], c);
}
__device__ __forceinline__ void mma(f32x4& c, const Planes2& a, const Planes3& b) {   // without the 2^-25 of both lowest terms
  c = mfma_bf(a.p[0], b.p[2], c);
  c = mfma_bf(a.p[1], b.p[1], c);
  c = mfma_bf(a.p[1], b.p[0], c);
  c = mfma_bf(a.p[0], b.p[1], c);
  c = mfma_bf(a.p[0], b.p[0], c);
}
__device__ __forceinline__ void mma(f32x4& c, const Planes3& a, const Planes3& b) {   // without the three terms below 2^-23
  c = mfma_bf(a.p[2], b.p[0], c);
  c = mfma_bf(a.p[0], b.p[2], c);
  c = mfma_bf(a.p[1], b.p[1], c);
  c = mfma_bf(a.p[1], b.p[0], c);
  c = mfma_bf(a.p[0], b.p[1], c);
  c = mfma_bf(a.p[0], b.p[0], c);
}

template <typename T> struct El;
template <> struct El<float> {
  static constexpr int C = 32, PLANES = 3;
  typedef Planes3 Raw; typedef Planes3 In; typedef Planes3 De; typedef Planes3 Wt;
  static __device__ __forceinline__ In in(const Raw& r) { return r; }
  static __device__ __forceinline__ De de(const f32x8& x) { return split3(x); }
  static __device__ __forceinline__ Wt wt(const f32x8& x) { return split3(x); }
  static __device__ __forceinline__ f32x8 wide(const Raw& r) {               // the exact sum again
    f32x8 x;
    const u32x4 h = __builtin_bit_cast(u32x4, r.p[0]), m = __builtin_bit_cast(u32x4, r.p[1]), l = __builtin_bit_cast(u32x4, r.p[2]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = half_lo(h[e]) + (half_lo(m[e]) + half_lo(l[e]));
      x[2 * e + 1] = half_hi(h[e]) + (half_hi(m[e]) + half_hi(l[e]));
    }
    return x;
  }
  static __device__ __forceinline__ void score(f32x4& c, const Raw& a, const Raw& b) { mma(c, a, b); }
};
template <> struct El<__bf16> {
  static constexpr int C = 64, PLANES = 1;
  typedef bf16x8 Raw; typedef Planes1 In; typedef Planes2 De; typedef Planes3 Wt;
  static __device__ __forceinline__ In in(const Raw& r) { return Planes1{{r}}; }
  static __device__ __forceinline__ De de(const f32x8& x) { return split2(x); }
  static __device__ __forceinline__ Wt wt(const f32x8& x) { return split3(x); }
  static __device__ __forceinline__ f32x8 wide(const Raw& r) {
    const u32x4 w = __builtin_bit_cast(u32x4, r);
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[2 * e] = half_lo(w[e]); x[2 * e + 1] = half_hi(w[e]); }
    return x;
  }
  static __device__ __forceinline__ void score(f32x4& c, const Raw& a, const Raw& b) { c = mfma_bf(a, b, c); }
};
template <> struct El<_Float16> {
  static constexpr int C = 64, PLANES = 1;
  typedef f16x8 Raw; typedef Planes2 In; typedef Planes2 De; typedef Planes3 Wt;
  static __device__ __forceinline__ f32x8 wide(const Raw& r) { return __builtin_convertvector(r, f32x8); }
  static __device__ __forceinline__ In in(const Raw& r) { return split2(wide(r)); }   // 11 significant bits: the two terms are exact
  static __device__ __forceinline__ De de(const f32x8& x) { return split2(x); }
  static __device__ __forceinline__ Wt wt(const f32x8& x) { return split3(x); }
  static __device__ __forceinline__ void score(f32x4& c, const Raw& a, const Raw& b) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ f32x8 join(const f32x4 a, const f32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// q and k lie in LDS with the columns of every 32 in the order of the fragments, column (half, q, j) = 16 half + 4 q + j at place
// 8 q + 4 half + j: a lane's {4g.., 16+4g..} are then neighbours.
__device__ __forceinline__ constexpr int place4(int c4) { return (c4 & ~7) * 4 + 8 * (c4 & 3) + 4 * ((c4 >> 2) & 1); }   // of the four columns from 4 c4

// row `row` of q or k, reduction indices 32 s + {4g..4g+3, 16+4g..16+4g+3}; `tile` has PITCH bytes a row and C rows a plane
template <typename T, int PITCH>
__device__ __forceinline__ typename El<T>::Raw row_frag(const char* tile, int row, int s, int g) {
  const char* a = tile + row * PITCH + (32 * s + 8 * g) * 2;
  if constexpr (El<T>::PLANES == 3) {
    Planes3 r;
#pragma unroll
    for (int q = 0; q < 3; ++q) r.p[q] = *reinterpret_cast<const bf16x8*>(a + q * El<T>::C * PITCH);
    return r;
  } else return __builtin_bit_cast(typename El<T>::Raw, *reinterpret_cast<const u32x4*>(a));
}
// column col0 + lane % 16 (col0 a multiple of 16), tokens 32 s + {4g.., 16+4g..}.  The whole wave takes part.
template <int PITCH> __device__ __forceinline__ u32x4 transposed(const char* a) {
  typedef s16x4 __attribute__((address_space(3))) * lds_p;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + 16 * PITCH));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
template <typename T, int PITCH, bool PLACED>
__device__ __forceinline__ typename El<T>::Raw col_frag(const char* tile, int s, int col0, int lane) {
  // each lane names 8 bytes of a 4 x 16 block (row lane % 16 / 4, columns 4 (lane % 4)..); lane l gets column l of the block
  const int c = PLACED ? place4(col0 / 4 + (lane & 3)) : col0 + 4 * (lane & 3);
  const char* a = tile + (32 * s + 4 * (lane >> 4) + ((lane >> 2) & 3)) * PITCH + c * 2;
  if constexpr (El<T>::PLANES == 3) {
    Planes3 r;
#pragma unroll
    for (int q = 0; q < 3; ++q) r.p[q] = __builtin_bit_cast(bf16x8, transposed<PITCH>(a + q * El<T>::C * PITCH));
    return r;
  } else return __builtin_bit_cast(typename El<T>::Raw, transposed<PITCH>(a));
}

// largest exponent pattern among the elements of a 16-byte unit, kept as a running maximum
template <typename T> struct Peak;
template <> struct Peak<float> {
  unsigned m = 0;
  __device__ __forceinline__ void see(const u32x4 w) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, w[e] & 0x7fffffffu);
  }
  __device__ __forceinline__ bool wild() const { return m >= 0x7f7f8000u; }   // infinite already as a bf16 term
};
template <unsigned short INF> struct Peak16 {
  u16x2 m = {0, 0};
  __device__ __forceinline__ void see(const u32x4 w) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
  }
  __device__ __forceinline__ bool wild() const { return m[0] >= INF || m[1] >= INF; }
};
template <> struct Peak<__bf16> : Peak16<0x7f80> {};
template <> struct Peak<_Float16> : Peak16<0x7c00> {};

template <typename T> __device__ __forceinline__ void store4(T* p, const f32x4 x, int valid, bool vec) {
  if (vec) {
    if (valid > 0) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = x;
      else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4*>(p) = __builtin_convertvector(x, t4);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < valid) p[r] = (T)x[r];
  }
}

// A [C][W] tile of tokens t .. t+n-1, columns c0 .. c0+W-1 (zero beyond `dim` and n): 16-byte units, unit u of a thread in its
// registers between the load and the write to LDS.
template <typename T, int C, int W, int NTH, bool PLACED>
struct Stage {
  static constexpr int E = 16 / (int)sizeof(T), UPR = W / E, UNITS = C * UPR, U = UNITS / NTH, PITCH = W * 2 + 16, ROWS = NTH / UPR, BYTES = C * PITCH * El<T>::PLANES;
  static_assert(UNITS % NTH == 0 && NTH % UPR == 0, "whole units per thread, whole rows per pass");
  u32x4 r[U];
  // p: the thread's first unit at the chunk's first token; its others lie ROWS tokens apart in the same columns, of which `cols` are
  // inside the row.  Addresses need only the element's alignment.
  template <bool FULL> __device__ __forceinline__ void load(const T* __restrict__ p, int64_t step, int n, int cols, int dim, int tid) {
    const int row = tid / UPR;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if (row + ROWS * i < n && (FULL || cols > 0)) {          // row < n <= C also keeps the unit inside the tile
        const T* q = p + step * (ROWS * i);
        if constexpr (FULL) w = *reinterpret_cast<const u32x4*>(q);
        else if (dim >= E) __builtin_memcpy(&w, q - (cols < E ? E - cols : 0), 16);   // a row's last, cut unit: the 16 bytes that end
        else {                                                                         // with the row, moved down when they are used
          for (int e = 0; e < cols; ++e) {
            if constexpr (sizeof(T) == 4) w[e] = __builtin_bit_cast(unsigned, q[e]);
            else w[e / 2] |= (unsigned)__builtin_bit_cast(unsigned short, q[e]) << (16 * (e & 1));
          }
        }
      }
      r[i] = w;
    }
  }
  static __device__ __forceinline__ u32x4 down(const u32x4 w, int bits) {   // 0 < bits < 128
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    u64x2 v = __builtin_bit_cast(u64x2, w);
    if (bits >= 64) { v[0] = v[1]; v[1] = 0; bits -= 64; }
    if (bits) { v[0] = v[0] >> bits | v[1] << (64 - bits); v[1] >>= bits; }
    return __builtin_bit_cast(u32x4, v);
  }
  template <bool FULL> __device__ __forceinline__ void store(char* tile, int cols, int dim, int tid, Peak<T>& peak) {
    const int over = !FULL && dim >= E && cols > 0 && cols < E ? (E - cols) * (int)sizeof(T) * 8 : 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (!FULL && over) r[i] = down(r[i], over);
      peak.see(r[i]);
      char* q = tile + (tid / UPR + ROWS * i) * PITCH;
      const int cu = tid % UPR;
      if constexpr (sizeof(T) == 4) {                // three exact bf16 terms, a plane each
        const Planes3 x = split3(__builtin_bit_cast(f32x8, __builtin_shufflevector(r[i], r[i], 0, 1, 2, 3, 0, 1, 2, 3)));
        q += (PLACED ? place4(cu) : 4 * cu) * 2;
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(q + k * C * PITCH) = __builtin_shufflevector(__builtin_bit_cast(u32x4, x.p[k]), u32x4{}, 0, 1);
      } else if constexpr (!PLACED) *reinterpret_cast<u32x4*>(q + cu * 16) = r[i];
      else {
        *reinterpret_cast<u32x2*>(q + place4(2 * cu) * 2) = u32x2{r[i][0], r[i][1]};
        *reinterpret_cast<u32x2*>(q + place4(2 * cu + 1) * 2) = u32x2{r[i][2], r[i][3]};
      }
    }
  }
};

// DP: both widths padded; STATE: only the segment's own contribution to the state; FULL: both widths are DP and all rows lie on 16-byte
// addresses.  Full widths of 64 are held to 168 registers for a third wave on each SIMD (16384 sequences of 32 tokens, bf16: gradient
// 272 us, 309 with two; 32768, fp32: forward 351 and 369, gradient 924 and 904).
template <typename T, int DP, bool STATE, bool FULL>
__global__ __launch_bounds__(DP / 16 * 64, DP == 64 && FULL && !STATE ? 3 : 2) void scan_kernel(const ScanP p) {
  typedef El<T> X;
  typedef typename X::Raw Raw;
  typedef typename X::In In;
  typedef typename X::De De;
  constexpr int C = X::C, WAVES = DP / 16, NTH = WAVES * 64;
  constexpr int KT = DP / 16, KS = DP / 32, CT = C / 16, JS = C / 32;
  typedef Stage<T, C, DP, NTH, true> SQ;
  typedef Stage<T, C, DP, NTH, false> SV;
  __shared__ __attribute__((aligned(16))) char lq[STATE ? 16 : SQ::BYTES];
  __shared__ __attribute__((aligned(16))) char lk[SQ::BYTES];
  __shared__ __attribute__((aligned(16))) char lv[SV::BYTES];
  __shared__ __attribute__((aligned(16))) float wj[C];   // per token of the chunk: weight of its k v^T in the state after the chunk,
  __shared__ float pw[C + 1];                            // lambda^n
  __shared__ float rj[C];                                // weight of the state on entry in its output (0: a reset lies between),
  __shared__ __attribute__((aligned(16))) int seg[C];    // number of resets before it reads
  __shared__ int wild[2];

  const Role& R = p.role[blockIdx.z];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
  const int split = blockIdx.y, t0 = split * p.seg, t1 = min(p.T, t0 + p.seg);
  const int bh = blockIdx.x;
  const int h = bh % p.H, cw = wave * 16;                 // first value column of the wave
  const double l2 = log2_decay(p.log_decay, h);
  const int off = R.off, dq = FULL ? DP : R.dq, dv = FULL ? DP : R.dv;
  // the thread's first unit of each operand: column and token offset are its own, the rest is the block's
  const int cq = (tid % SQ::UPR) * SQ::E, cv = (tid % SV::UPR) * SV::E, nq = dq - cq, nv = dv - cv;
  const int64_t ql = (tid / SQ::UPR) * R.qs[1] + cq, kl = (tid / SQ::UPR) * R.ks[1] + cq, vl = (tid / SV::UPR) * R.vs[1] + cv;
  const int64_t sz = (int64_t)dq * dv;

  SQ sq, sk;
  SV sv;
  int rbyte = 0;
  auto fetch = [&](int bh, int t, int n) {
    const int64_t b = bh / p.H;
    if constexpr (!STATE) sq.template load<FULL>(static_cast<const T*>(R.q) + b * R.qs[0] + h * R.qs[2] + t * R.qs[1] + ql, R.qs[1], n, nq, dq, tid);
    sk.template load<FULL>(static_cast<const T*>(R.k) + b * R.ks[0] + h * R.ks[2] + t * R.ks[1] + kl, R.ks[1], n, nq, dq, tid);
    sv.template load<FULL>(static_cast<const T*>(R.v) + b * R.vs[0] + h * R.vs[2] + t * R.vs[1] + vl, R.vs[1], n, nv, dv, tid);
    rbyte = (R.resets && lane < n) ? R.resets[b * R.rs[0] + (t + lane) * R.rs[1]] : 0;
  };
  auto load_state = [&](int bh, f32x4 (&S)[KT]) {
    const float* s0 = nullptr;
    int sr = R.s_row, sc = R.s_col;
    if (!STATE) {
      if (split == 0) s0 = R.s0 ? R.s0 + bh * sz : nullptr;
      else { s0 = p.ws + R.ws + ((int64_t)(split - 1) * p.BH + bh) * sz; sr = dv; sc = 1; }
    }
    if (FULL && s0 && sr == 1) {                          // transposed: a lane's four rows are neighbours
      typedef f32x4 __attribute__((aligned(4))) unit;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) S[kt] = *reinterpret_cast<const unit*>(s0 + (unsigned)((cw + m) * sc + 16 * kt + 4 * g));
      return;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * kt + 4 * g + r, col = cw + m;
        S[kt][r] = (s0 && row < dq && col < dv) ? s0[(unsigned)(row * sr + col * sc)] : 0.0f;
      }
  };
  auto store_state = [&](int bh, const f32x4 (&S)[KT]) {
    float* s1 = nullptr;
    int sr = R.s_row, sc = R.s_col;
    if (STATE) { s1 = p.ws + R.ws + ((int64_t)split * p.BH + bh) * sz; sr = dv; sc = 1; }
    else if (split == p.n_splits - 1) s1 = R.s1 ? R.s1 + bh * sz : nullptr;
    if (!s1) return;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * kt + 4 * g + r, col = cw + m;
        if (row < dq && col < dv) s1[(unsigned)(row * sr + col * sc)] = S[kt][r];
      }
  };
  int t = t0, n = min(C, t1 - t0);
  if (n > 0) fetch(bh, t, n);
  f32x4 S[KT];
  load_state(bh, S);
  // lambda^n for every distance inside a chunk; scores weigh by lambda^(i-j): inside a diagonal tile directly, between tiles d + 1 apart
  // as lambda^(16 d + m + 1) * lambda^(15 - (4g + r)), both exponents non-negative
  for (int i = tid; i <= C; i += NTH) pw[i] = decay_pow(l2, i);
  if (tid < 2) wild[tid] = 0;
  __syncthreads();
  const float scale = R.wscale * R.oscale, pC = pw[C];
  float ai[CT], bj[4], dg[4];
  if constexpr (!STATE) {
#pragma unroll
    for (int i = 0; i + 1 < CT; ++i) ai[i] = pw[16 * i + m + 1] * scale;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      bj[r] = pw[15 - (4 * g + r)];
      dg[r] = pw[max(m - (4 * g + r), 0)] * scale;
    }
  }
  int plain_n = 0;                                        // length of the chunk without resets that the tables stand for
  int any_reset = 0, careful = t0, turn = 0;

  while (t < t1) {
    // ---- stage the chunk
    const uint64_t rm = __ballot(rbyte != 0);
    if (rm != 0 || plain_n != n) {
      if (tid < C) {
        const uint64_t mj = (off ? (2ull << tid) : (1ull << tid)) - 1;
        wj[tid] = (tid < n && (rm & ~mj) == 0) ? pw[max(n - off - tid, 0)] * R.wscale : 0.0f;
        if constexpr (!STATE) {
          rj[tid] = (rm & mj) == 0 ? pw[tid + off] * R.oscale : 0.0f;
          seg[tid] = __builtin_popcountll(rm & mj);
        }
      }
      plain_n = rm ? 0 : n;
    }
    Peak<T> peak;
    if constexpr (!STATE) sq.template store<FULL>(lq, nq, dq, tid, peak);
    sk.template store<FULL>(lk, nq, dq, tid, peak);
    sv.template store<FULL>(lv, nv, dv, tid, peak);
    if (peak.wild()) wild[turn] = 1;
    __syncthreads();
    const bool found = wild[turn] != 0;
    if (tid == 0) wild[turn ^ 1] = 0;
    turn ^= 1;
    if (found && n > 1) {                               // walk these tokens one at a time
      careful = t + n;
      n = 1;
      __syncthreads();
      fetch(bh, t, n);
      continue;
    }
    const int tn = t + n, nn = tn < careful ? 1 : min(C, t1 - tn);
    if (tn < t1) fetch(bh, tn, nn);

    // ---- the chunk's products (none for a wave whose columns are padding)
    if (cw < dv) {
    if constexpr (!STATE) {
      De sf[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) sf[s] = X::de(join(S[2 * s], S[2 * s + 1]));
      In vin[JS];
#pragma unroll
      for (int s = 0; s < JS; ++s) vin[s] = X::in(col_frag<T, SV::PITCH, false>(lv, s, cw, lane));
      const int64_t obase = (int64_t)(bh / p.H) * R.os[0] + h * R.os[2];
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        if (16 * it >= n) break;
        if constexpr (X::PLANES == 3) asm volatile("" ::: "memory");   // and again for every 16 rows, not kept in registers
        Raw qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = row_frag<T, SQ::PITCH>(lq, 16 * it + m, s, g);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if (32 * s >= dq) break;
          mma(o, sf[s], X::in(qf[s]));
        }
        const int i = 16 * it + m;
        const float rd = rj[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = rd != 0.0f ? o[r] * rd : 0.0f;
#pragma unroll
        for (int s = 0; s < JS; ++s) {
          if (2 * s > it) break;
          f32x4 pt[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int jt = 2 * s + u;
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
            if (jt <= it) {
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) {
                if constexpr (X::PLANES == 3) asm volatile("" ::: "memory");   // three planes: fragments are read as they are needed
                if (32 * ks < dq) X::score(a, row_frag<T, SQ::PITCH>(lk, 16 * jt + m, ks, g), qf[ks]);
              }
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                if (jt == it) a[r] = m >= 4 * g + r ? a[r] * dg[r] : 0.0f;
                else a[r] = a[r] * (ai[it - jt - 1] * bj[r]);
              }
              if (rm) {
                const int si = seg[i];
#pragma unroll
                for (int r = 0; r < 4; ++r) a[r] = seg[16 * jt + 4 * g + r] == si ? a[r] : 0.0f;
              }
            }
            pt[u] = a;
          }
          const De pf = X::de(join(pt[0], pt[1]));
          mma(o, vin[s], pf);
        }
        if (i < n) {
          const int c = cw + 4 * g;
          store4<T>(static_cast<T*>(R.out) + obase + (t + i) * R.os[1] + c, o, dv - c, (dv & 3) == 0);
        }
      }
    }
    // ---- the state after the chunk
    if constexpr (X::PLANES == 3) asm volatile("" ::: "memory");
    const float dec = n == C ? pC : pw[n];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[kt][r] = rm ? 0.0f : S[kt][r] * dec;
#pragma unroll
    for (int s = 0; s < JS; ++s) {
      if (32 * s >= n || (n == 1 && rm && !off)) break;   // a lone token whose write its own reset drops: zero times an infinity is none
      const f32x8 w = join(*reinterpret_cast<const f32x4*>(wj + 32 * s + 4 * g), *reinterpret_cast<const f32x4*>(wj + 32 * s + 16 + 4 * g));
      const typename X::Wt vw = X::wt(X::wide(col_frag<T, SV::PITCH, false>(lv, s, cw, lane)) * w);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if (16 * kt >= dq) break;
        mma(S[kt], X::in(col_frag<T, SQ::PITCH, true>(lk, s, 16 * kt, lane)), vw);
      }
    }
    }
    any_reset |= rm != 0;
    __syncthreads();                                     // every wave has read the tiles
    t = tn;
    n = nn;
  }
  store_state(bh, S);
  if (STATE && tid == 0) p.flags[((int64_t)blockIdx.z * p.n_splits + split) * p.BH + bh] = any_reset;
}

// Between the two passes over a split sequence: the segments' own contributions become the states on entry.  Slot s holds segment
// s's contribution before and the state on entry of segment s + 1 after; every element walks the segments by itself.
__global__ __launch_bounds__(256) void prefix_kernel(const ScanP p) {
  const Role& R = p.role[blockIdx.z];
  const int bh = blockIdx.y, h = bh % p.H;
  const int64_t sz = (int64_t)R.dq * R.dv;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= sz) return;
  const int row = (int)(e / R.dv), col = (int)(e % R.dv);
  float E = R.s0 ? R.s0[bh * sz + (int64_t)row * R.s_row + (int64_t)col * R.s_col] : 0.0f;
  const float dec = decay_pow(log2_decay(p.log_decay, h), p.seg);   // every segment but the last is whole
  float* w = p.ws + R.ws + bh * sz + e;
  const int* f = p.flags + (int64_t)blockIdx.z * p.n_splits * p.BH + bh;
  const int64_t step = (int64_t)p.BH * sz;
  const int last = p.n_splits - 1;
  constexpr int AHEAD = 8;
  for (int s = 0; s < last; s += AHEAD) {
    float L[AHEAD];
    int fl[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      L[a] = s + a < last ? w[(s + a) * step] : 0.0f;
      fl[a] = s + a < last ? f[(int64_t)(s + a) * p.BH] : 0;
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
      if (s + a < last) {
        E = (fl[a] ? 0.0f : E * dec) + L[a];
        w[(s + a) * step] = E;
      }
  }
}

// One token per row: S <- lambda S + k v^T in place, o = scale S^T q.  One block per (row, head); a thread owns VEC neighbouring
// columns and every RG-th row of S.  Bound by the state's read and write: 8192 rows of 4 heads, 64 x 64: 205 us for 1.11 GB, 5.4 TB/s.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void step_kernel(const mrl_attention a, float* __restrict__ state, T* __restrict__ out, int ncp) {
  __shared__ float kq[2][MRL_ATTENTION_MAX_DIM];
  __shared__ __attribute__((aligned(16))) float red[256 * VEC];
  const int tid = threadIdx.x, bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads;
  const int K = a.dim_k, V = a.dim_v;
  const int c = (tid % ncp) * VEC, rg = tid / ncp, RG = 256 / ncp;
  const bool clear = a.resets && a.resets[b] != 0;
  const float dec = decay_pow(log2_decay(a.log_decay, h), 1);
  if (tid < K) {
    kq[0][tid] = (float)(static_cast<const T*>(a.k) + b * a.k_stride[0] + h * a.k_stride[2])[tid];
    kq[1][tid] = (float)(static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[2])[tid];
  }
  float v[VEC], o[VEC];
  const T* vp = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    v[e] = c + e < V ? (float)vp[c + e] : 0.0f;
    o[e] = 0.0f;
  }
  float* s = state + (int64_t)bh * K * V + c;
  __syncthreads();
  if (c < V) {
    constexpr int UN = 4;
    for (int r0 = rg; r0 < K; r0 += RG * UN) {
      typedef float fv __attribute__((ext_vector_type(VEC)));
      fv x[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int r = r0 + u * RG;
        x[u] = (!clear && r < K) ? *reinterpret_cast<const fv*>(s + (int64_t)r * V) * dec : fv(0.0f);
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int r = r0 + u * RG;
        if (r < K) {
          const float kr = kq[0][r], qr = kq[1][r];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            x[u][e] = __builtin_fmaf(kr, v[e], x[u][e]);
            o[e] = __builtin_fmaf(qr, x[u][e], o[e]);
          }
          *reinterpret_cast<fv*>(s + (int64_t)r * V) = x[u];
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) red[rg * ncp * VEC + c + e] = o[e];
  __syncthreads();
  if (tid < V) {
    float sum = 0.0f;
    for (int r = 0; r < RG; ++r) sum += red[r * ncp * VEC + tid];
    out[((int64_t)b * a.heads + h) * V + tid] = (T)(sum * a.scale);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
struct Plan { int dp, seg, n_splits; };

int chunk_of(int dtype) { return dtype == MRL_F32 ? El<float>::C : El<__bf16>::C; }

int check(const mrl_attention* p, const char* what) {
  if (!p) MEM_FAIL(MRL_EINVAL, "%s: null description", what);
  if (p->dtype < MRL_F32 || p->dtype > MRL_F16) MEM_FAIL(MRL_EINVAL, "%s: dtype %d (float32, bfloat16 or float16)", what, p->dtype);
  if (p->batch < 0 || p->steps < 0 || p->heads < 1) MEM_FAIL(MRL_EINVAL, "%s: batch %lld, steps %lld, heads %d", what, (long long)p->batch, (long long)p->steps, p->heads);
  if (p->dim_k < 1 || p->dim_k > MRL_ATTENTION_MAX_DIM || p->dim_v < 1 || p->dim_v > MRL_ATTENTION_MAX_DIM)
    MEM_FAIL(MRL_EINVAL, "%s: dim_k %d, dim_v %d (1..%d each)", what, p->dim_k, p->dim_v, MRL_ATTENTION_MAX_DIM);
  if (p->steps >= (int64_t(1) << 30)) MEM_FAIL(MRL_EINVAL, "%s: %lld steps", what, (long long)p->steps);
  // one block each, and a grid has less than 2^32 threads: 256 of them stepping, up to 512 of a wide scan
  if (p->batch >= (int64_t(1) << 23) / p->heads) MEM_FAIL(MRL_EINVAL, "%s: %lld batch rows x %d heads (below 2^23)", what, (long long)p->batch, p->heads);
  return MRL_OK;
}

// outputs are stored in units of up to 16 bytes
bool on_units(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if ((uintptr_t)q & 15) return false;
  return true;
}

int check_pointers(const mrl_attention* p, const char* what) {
  if (p->batch == 0) return MRL_OK;
  if (!p->log_decay) MEM_FAIL(MRL_EINVAL, "%s: null log_decay", what);
  if (p->steps > 0 && (!p->q || !p->k || !p->v)) MEM_FAIL(MRL_EINVAL, "%s: null q, k or v", what);
  return MRL_OK;
}

// How the work is cut.  A block has one wave for every 16 value columns.  Where there are blocks for every CU and waves for every SIMD,
// one walks over all its tokens: 272 blocks of 64 x 64, 655 tokens, take 88 us in fp32 and 47 in bf16, split in two 115 and 69.  With
// fewer the tokens are split into segments of whole chunks, whose states are computed first, joined, and handed to the second pass,
// 2048 waves in all (two a SIMD): 8 blocks of 128 x 128, 16384 tokens, bf16, take 86 us so, 134 with half as many waves and 102 with twice.
Plan plan_of(const mrl_attention* p, int roles) {
  Plan r;
  const int d = std::max(p->dim_k, p->dim_v);
  r.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128;
  const int C = chunk_of(p->dtype);
  const int64_t blocks = std::max<int64_t>(1, p->batch * p->heads * roles);
  const int64_t chunks = cdiv(p->steps, C);
  const int waves = r.dp / 16;
  int64_t splits = blocks >= std::max(256, 1024 / waves) ? 1 : std::max<int64_t>(1, std::min<int64_t>(cdiv(2048 / waves, blocks), chunks));
  const int64_t per = std::max<int64_t>(1, cdiv(chunks, splits));
  r.seg = (int)(per * C);
  r.n_splits = (int)std::max<int64_t>(1, cdiv(chunks, per));
  return r;
}

int64_t role_floats(const mrl_attention* p, const Plan& pl) {
  return pl.n_splits > 1 ? (int64_t)(pl.n_splits - 1) * p->batch * p->heads * p->dim_k * p->dim_v : 0;
}
int64_t ws_bytes(const mrl_attention* p, const Plan& pl, int roles) {
  if (pl.n_splits <= 1) return 0;
  return role_floats(p, pl) * roles * 4 + (int64_t)roles * pl.n_splits * p->batch * p->heads * 4;
}

template <typename T, int DP, bool FULL> void launch_as(const ScanP& a, const Plan& pl, int roles, hipStream_t st) {
  const unsigned nth = DP / 16 * 64;
  if (pl.n_splits > 1) {
    hipLaunchKernelGGL((scan_kernel<T, DP, true, FULL>), dim3(a.BH, pl.n_splits - 1, roles), dim3(nth), 0, st, a);
    const int64_t sz = (int64_t)a.role[0].dq * a.role[0].dv;
    hipLaunchKernelGGL(prefix_kernel, dim3((unsigned)cdiv(sz, 256), a.BH, roles), dim3(256), 0, st, a);
  }
  hipLaunchKernelGGL((scan_kernel<T, DP, false, FULL>), dim3(a.BH, pl.n_splits, roles), dim3(nth), 0, st, a);
}
template <typename T> void launch(const ScanP& a, const Plan& pl, int roles, hipStream_t st) {
  bool full = true;
  for (int i = 0; i < roles; ++i) full = full && a.role[i].vec && a.role[i].dq == pl.dp && a.role[i].dv == pl.dp;
  auto go = [&](auto v) {
    constexpr bool FULL = decltype(v)::value;
    if (pl.dp == 32) launch_as<T, 32, FULL>(a, pl, roles, st);
    else if (pl.dp == 64) launch_as<T, 64, FULL>(a, pl, roles, st);
    else if (pl.dp == 96) launch_as<T, 96, FULL>(a, pl, roles, st);
    else launch_as<T, 128, FULL>(a, pl, roles, st);
  };
  if (full) go(std::true_type());
  else go(std::false_type());
}
int dispatch(const mrl_attention* p, ScanP& a, const Plan& pl, int roles, void* ws, int64_t bytes, void* stream, const char* what) {
  const int64_t need = ws_bytes(p, pl, roles);
  if (need > 0 && (!ws || bytes < need)) MEM_FAIL(MRL_ENOSPC, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes, (long long)need);
  if (need > 0 && ((uintptr_t)ws & 15)) MEM_FAIL(MRL_EINVAL, "%s: workspace is not aligned", what);
  a.log_decay = p->log_decay;
  a.T = (int)p->steps; a.seg = pl.seg; a.n_splits = pl.n_splits; a.H = p->heads;
  a.BH = (int)(p->batch * p->heads);
  a.ws = static_cast<float*>(ws);
  for (int i = 0; i < roles; ++i) {
    a.role[i].ws = role_floats(p, pl) * i;
    a.role[i].vec = a.role[i].vec && on_units({a.role[i].s0});
  }
  a.flags = reinterpret_cast<int*>(a.ws + role_floats(p, pl) * roles);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == MRL_F32) launch<float>(a, pl, roles, st);
  else if (p->dtype == MRL_BF16) launch<__bf16>(a, pl, roles, st);
  else launch<_Float16>(a, pl, roles, st);
  MEM_CHECK_LAUNCH(what);
  return MRL_OK;
}

struct Operand { const void* p; const int64_t* s; };

// 16-byte addresses: the first one, and every stride that is used
bool whole(const Operand& o, int dim, int es, const mrl_attention* p) {
  const int e = 16 / es;
  return dim % e == 0 && ((uintptr_t)o.p & 15) == 0 && (p->batch == 1 || o.s[0] % e == 0) && (p->steps <= 1 || o.s[1] % e == 0) && (p->heads == 1 || o.s[2] % e == 0);
}

void set_role(Role& r, const mrl_attention* p, bool back, const Operand& q, const Operand& k, const Operand& v, int dq, int dv, void* out) {
  const int es = p->dtype == MRL_F32 ? 4 : 2;
  const int64_t last = back ? p->steps - 1 : 0, sign = back ? -1 : 1;
  auto put = [&](const void*& dst, int64_t* ds, const Operand& o) {
    ds[0] = o.s[0]; ds[1] = sign * o.s[1]; ds[2] = o.s[2];
    dst = static_cast<const char*>(o.p) + last * o.s[1] * es;
  };
  put(r.q, r.qs, q); put(r.k, r.ks, k); put(r.v, r.vs, v);
  r.os[2] = dv; r.os[0] = p->steps * p->heads * (int64_t)dv; r.os[1] = sign * p->heads * (int64_t)dv;
  r.out = out ? static_cast<char*>(out) + last * p->heads * (int64_t)dv * es : nullptr;
  r.resets = p->resets ? p->resets + last : nullptr;
  r.rs[0] = p->steps; r.rs[1] = sign;
  r.dq = dq; r.dv = dv; r.off = back ? 0 : 1;
  r.vec = whole(q, dq, es, p) && whole(k, dq, es, p) && whole(v, dv, es, p);
  r.oscale = r.wscale = 1.0f;
  r.s0 = nullptr; r.s1 = nullptr; r.s_row = dv; r.s_col = 1;
}

}  // namespace

extern "C" int64_t mrl_linear_attention_workspace_bytes(const mrl_attention* p, int32_t backward) {
  const int rc = check(p, "mrl_linear_attention_workspace_bytes");
  if (rc) return rc;
  const int roles = backward ? 3 : 1;
  return ws_bytes(p, plan_of(p, roles), roles);
}

extern "C" int mrl_linear_attention(const mrl_attention* p, void* out, float* final_state, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mrl_linear_attention";
  int rc = check(p, what);
  if (rc || (rc = check_pointers(p, what))) return rc;
  if (p->batch == 0) return MRL_OK;
  if (!final_state || (p->steps > 0 && !out)) MEM_FAIL(MRL_EINVAL, "%s: null output", what);
  if (!on_units({out})) MEM_FAIL(MRL_EINVAL, "%s: out is not aligned to 16 bytes", what);
  ScanP a;
  Role& r = a.role[0];
  set_role(r, p, false, {p->q, p->q_stride}, {p->k, p->k_stride}, {p->v, p->v_stride}, p->dim_k, p->dim_v, out);
  r.oscale = p->scale;
  r.s0 = p->initial_state;
  r.s1 = final_state;
  return dispatch(p, a, plan_of(p, 1), 1, workspace, workspace_bytes, stream, what);
}

extern "C" int mrl_linear_attention_backward(const mrl_attention* p, const void* d_out, const int64_t* d_out_stride_host, const float* d_final_state, void* dq,
                                             void* dk, void* dv, float* d_initial_state, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mrl_linear_attention_backward";
  int rc = check(p, what);
  if (rc || (rc = check_pointers(p, what))) return rc;
  if (p->batch == 0) return MRL_OK;
  if (p->steps > 0 && (!d_out || !d_out_stride_host)) MEM_FAIL(MRL_EINVAL, "%s: null d_out", what);
  if (p->steps > 0 && d_initial_state && !dv) MEM_FAIL(MRL_EINVAL, "%s: d_initial_state comes with dv", what);
  if (!on_units({dq, dk, dv})) MEM_FAIL(MRL_EINVAL, "%s: dq, dk and dv have to be aligned to 16 bytes", what);
  static const int64_t none[3] = {0, 0, 0};
  const Operand q{p->q, p->q_stride}, k{p->k, p->k_stride}, v{p->v, p->v_stride}, d{d_out, d_out_stride_host ? d_out_stride_host : none};
  const int K = p->dim_k, V = p->dim_v;
  ScanP a;
  int n = 0;
  if (dq) {                 // reads S transposed
    Role& r = a.role[n++];
    set_role(r, p, false, d, v, k, V, K, dq);
    r.oscale = p->scale;
    r.s0 = p->initial_state;
    r.s_row = 1; r.s_col = V;
  }
  // dk, dv: the state is the gradient of S (transposed for dk); scale belongs to every q do^T but not to d_final_state
  if (dk) {
    Role& r = a.role[n++];
    set_role(r, p, true, v, d, q, V, K, dk);
    r.wscale = p->scale;
    r.s0 = d_final_state;
    r.s_row = 1; r.s_col = V;
  }
  if (dv || d_initial_state) {
    Role& r = a.role[n++];
    set_role(r, p, true, k, q, d, K, V, dv);
    r.wscale = p->scale;
    r.s0 = d_final_state;
    r.s1 = d_initial_state;
  }
  if (n == 0) return MRL_OK;
  return dispatch(p, a, plan_of(p, 3), n, workspace, workspace_bytes, stream, what);
}

extern "C" int mrl_linear_attention_step(const mrl_attention* p, float* state, void* out, void* stream) {
  const char* what = "mrl_linear_attention_step";
  int rc = check(p, what);
  if (rc || (rc = check_pointers(p, what))) return rc;
  if (p->steps != 1) MEM_FAIL(MRL_EINVAL, "%s: %lld steps, one is meant", what, (long long)p->steps);
  if (p->batch == 0) return MRL_OK;
  if (!state || !out) MEM_FAIL(MRL_EINVAL, "%s: null state or output", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool vec = p->dim_v % 4 == 0 && ((uintptr_t)state & 15) == 0;
  int ncp = 1;
  while (ncp * (vec ? 4 : 1) < p->dim_v) ncp *= 2;
  const dim3 grid((unsigned)(p->batch * p->heads)), block(256);
  auto run = [&](auto tag) {
    typedef decltype(tag) T;
    if (vec) hipLaunchKernelGGL((step_kernel<T, 4>), grid, block, 0, st, *p, state, static_cast<T*>(out), ncp);
    else hipLaunchKernelGGL((step_kernel<T, 1>), grid, block, 0, st, *p, state, static_cast<T*>(out), ncp);
  };
  if (p->dtype == MRL_F32) run(0.0f);
  else if (p->dtype == MRL_BF16) run((__bf16)0.0f);
  else run((_Float16)0.0f);
  MEM_CHECK_LAUNCH(what);
  return MRL_OK;
}
