// Group norm with an activation on channels-last data for gfx950, forward and backward:
//   xhat = (x - mean_ng) rstd_ng,  z = xhat w_c + b_c,  y = act(z)
//   dz = dy act'(z),  dw_c = sum dz xhat,  db_c = sum dz,  dx = rstd (w dz - m1 - xhat m2),  m1 = mean_g(w dz), m2 = mean_g(w dz xhat)
// Bound by memory: forward one read and one write of the data, backward two reads and one write.  65536 rows of 512 channels in 8
// groups, bf16, SiLU: forward 32 us (4.2 TB/s), backward 44 us (4.6 TB/s) and 4 for the parameters; 64 x 7056 pixels of 32 channels,
// fp32: 34 us forward and 60 backward for 289 MB in all.  Two shapes of it:
//   * one pixel per sample (tokens): a group is one contiguous run of channels, held in the registers of a team of lanes; one pass.
//     Teams keep their group while they walk over the samples, so the parameters are read once and their gradients add up in
//     registers; a last launch adds the teams' sums.
//   * many pixels: blocks take runs of pixels with all (up to 256 vectors of) channels, a thread always the same ones.  The first
//     launch leaves count, mean and sum of squares of its part, the second joins the parts and writes y; backwards the first
//     leaves the two sums of each channel, a small one joins them, the third writes dx.  The second reading of x comes from the
//     256 MB cache behind the L2s where the data fit it.  Tokens whose group no team holds (over 256 vectors) come here too, one pixel
//     each: two readings, and backwards a workspace of 16 bytes a value (65536 x 4096 in one group, bf16: 1.0 ms forward, 3.8 backward).
// Means and variances are joined pairwise (count, mean, centred squares), so a large mean costs no digits.  The mean of equal values is
// their value, so that such a group has no spread (a spacing of the mean, divided by sqrt(eps), would show): of 16-bit values by exact
// sums and true quotients, of fp32 ones by taking off the mean of what the first mean leaves.  Every sum has one order: no atomics.
#include "memory_common.hip.h"

#include <type_traits>

using namespace mrl::mem;

namespace {

// Vectors of V elements of T as fp32; V divides the channels of a group, and rows start on V elements.
template <typename T, int V> struct Vec {
  typedef T tv __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ void load(const T* p, float (&x)[V]) {
    if constexpr (V == 1) x[0] = (float)*p;
    else {
      const tv r = *reinterpret_cast<const tv*>(p);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = (float)r[e];
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[V]) {
    if constexpr (V == 1) *p = (T)x[0];
    else {
      tv r;
#pragma unroll
      for (int e = 0; e < V; ++e) r[e] = (T)x[e];
      *reinterpret_cast<tv*>(p) = r;
    }
  }
};

// The same at any address, of which `left` elements belong to the row (the others read as zero and are not stored).
template <typename T, int V> struct Ragged {
  typedef T tv __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ void load(const T* p, int left, float (&x)[V]) {
    if (left >= V) {
      tv r;
      __builtin_memcpy(&r, p, sizeof(r));
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = (float)r[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = e < left ? (float)p[e] : 0.0f;
    }
  }
  static __device__ __forceinline__ void store(T* p, int left, const float (&x)[V]) {
    if (left >= V) {
      tv r;
#pragma unroll
      for (int e = 0; e < V; ++e) r[e] = (T)x[e];
      __builtin_memcpy(p, &r, sizeof(r));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) p[e] = (T)x[e];
    }
  }
};

struct GnP {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float *mean, *rstd;
  const float *cmean, *crstd;
  float* ws;
  int64_t N, L;
  int C, G, Cg, act, pdt;   // pdt: parameters are fp32
  float eps;
  int teams;                // token kernels: all teams of the launch, a multiple of G
  int splits, chunk;        // pixel kernels: parts of a sample, pixels of a part
  int cvs, slabs;           // channel vectors of a block, blocks that cover the channels
  int spg;                  // blocks that share a group (1, or more where a group has over 256 vectors)
};

template <typename T> __device__ __forceinline__ float param(const void* p, int pdt, int64_t c, float otherwise) {
  if (!p) return otherwise;
  return pdt ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
}
template <typename T> __device__ __forceinline__ void put_param(void* p, int pdt, int64_t c, float v) {
  if (pdt) static_cast<float*>(p)[c] = v;
  else static_cast<T*>(p)[c] = (T)v;
}

// sum over the TL lanes of a team (TL a power of two up to 64): every lane gets it.  Up to 16 lanes through the register file's own
// lane permutations (neighbours, pairs, then the halves of 8 and 16 mirrored, whose lanes hold equal sums by then), not through LDS.
template <int CTRL> __device__ __forceinline__ float lanes(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int TL> __device__ __forceinline__ float team_sum(float v) {
  if constexpr (TL >= 2) v += lanes<0xb1>(v);
  if constexpr (TL >= 4) v += lanes<0x4e>(v);
  if constexpr (TL >= 8) v += lanes<0x141>(v);
  if constexpr (TL >= 16) v += lanes<0x140>(v);
  if constexpr (TL >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (TL >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// A product as it is rounded: not to be fused into the difference that follows, which would be taken of another mean than is kept.
__device__ __forceinline__ float rounded(float x) {
  asm("" : "+v"(x));
  return x;
}

// ---- one pixel per sample --------------------------------------------------------------------------------------------------------
// Row r = n G + g is Cg contiguous values.  A team of TL lanes, NV vectors per lane, walks the rows team, team + teams, ... of its group.
// RAG: Cg is not a number of whole vectors, and rows lie on any address.
template <typename T, int V, int TL, int NV, bool RAG>
__global__ __launch_bounds__(256) void token_fwd_kernel(const GnP p) {
  const int lane = threadIdx.x % TL;
  const int team = blockIdx.x * (256 / TL) + threadIdx.x / TL;
  if (team >= p.teams) return;                              // whole teams leave: no lane of a team is missing from its sums
  const int g = team % p.G;
  const int64_t rows = p.N * p.G;
  const float inv = 1.0f / (float)p.Cg;
  float w[NV][V], b[NV][V];
  bool in[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + TL * i) * V;
    in[i] = c < p.Cg;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[i][e] = in[i] && (!RAG || c + e < p.Cg) ? param<T>(p.w, p.pdt, g * p.Cg + c + e, 1.0f) : 0.0f;
      b[i][e] = in[i] && (!RAG || c + e < p.Cg) ? param<T>(p.b, p.pdt, g * p.Cg + c + e, 0.0f) : 0.0f;
    }
  }
  auto left = [&](int i) { return p.Cg - (lane + TL * i) * V; };
  auto read = [&](const T* row, int i, float (&f)[V]) {
    if constexpr (RAG) Ragged<T, V>::load(row + (lane + TL * i) * V, left(i), f);
    else Vec<T, V>::load(row + (lane + TL * i) * V, f);
  };
  auto write = [&](T* row, int i, const float (&f)[V]) {
    if constexpr (RAG) Ragged<T, V>::store(row + (lane + TL * i) * V, left(i), f);
    else Vec<T, V>::store(row + (lane + TL * i) * V, f);
  };
  for (int64_t r = team; r < rows; r += p.teams) {
    const T* x = static_cast<const T*>(p.x) + r * p.Cg;
    T* y = static_cast<T*>(p.y) + r * p.Cg;
    float v[NV][V], s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (in[i]) {
        read(x, i, v[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) s += v[i][e];
      }
    // The sum of up to 2048 equal values of 16 bits is exact and its quotient their value; an fp32 mean is freed of its rounding by the
    // mean of what it leaves.
    float mean = sizeof(T) == 2 ? team_sum<TL>(s) / (float)p.Cg : rounded(team_sum<TL>(s) * inv);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (in[i]) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] -= mean;
      }
    if constexpr (sizeof(T) == 4) {
      float d = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (!RAG || e < left(i)) d += v[i][e];
        }
      d = team_sum<TL>(d) * inv;
      mean += d;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[i][e] -= d;
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (in[i]) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (!RAG || e < left(i)) q = __builtin_fmaf(v[i][e], v[i][e], q);
      }
    const float rstd = 1.0f / sqrtf(team_sum<TL>(q) * inv + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (in[i]) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = __builtin_fmaf(v[i][e] * rstd, w[i][e], b[i][e]);
        act_fwd<V>(p.act, v[i]);
        write(y, i, v[i]);
      }
    if (p.mean && lane == 0) {
      p.mean[r] = mean;
      p.rstd[r] = rstd;
    }
  }
}

// The teams' parameter sums go to ws as rows [2][C]: row team / G, or one row per block where its teams hold every group equally often.
template <typename T, int V, int TL, int NV, bool RAG>
__global__ __launch_bounds__(256) void token_bwd_kernel(const GnP p) {
  constexpr int TB = 256 / TL;
  __shared__ float red[2][V][256];
  const int lane = threadIdx.x % TL, lt = threadIdx.x / TL;
  const int team = blockIdx.x * TB + lt;
  const bool live = team < p.teams;
  const int g = team % p.G;
  const int64_t rows = p.N * p.G;
  const float inv = 1.0f / (float)p.Cg;
  float w[NV][V], b[NV][V], dw[NV][V], db[NV][V];
  bool in[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + TL * i) * V;
    in[i] = live && c < p.Cg;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[i][e] = in[i] && (!RAG || c + e < p.Cg) ? param<T>(p.w, p.pdt, g * p.Cg + c + e, 1.0f) : 0.0f;
      b[i][e] = in[i] && (!RAG || c + e < p.Cg) ? param<T>(p.b, p.pdt, g * p.Cg + c + e, 0.0f) : 0.0f;
      dw[i][e] = db[i][e] = 0.0f;
    }
  }
  auto left = [&](int i) { return p.Cg - (lane + TL * i) * V; };
  auto read = [&](const T* row, int i, float (&f)[V]) {
    if constexpr (RAG) Ragged<T, V>::load(row + (lane + TL * i) * V, left(i), f);
    else Vec<T, V>::load(row + (lane + TL * i) * V, f);
  };
  auto write = [&](T* row, int i, const float (&f)[V]) {
    if constexpr (RAG) Ragged<T, V>::store(row + (lane + TL * i) * V, left(i), f);
    else Vec<T, V>::store(row + (lane + TL * i) * V, f);
  };
  if (live) {
    for (int64_t r = team; r < rows; r += p.teams) {
      const T* x = static_cast<const T*>(p.x) + r * p.Cg;
      const T* dy = static_cast<const T*>(p.dy) + r * p.Cg;
      T* dx = static_cast<T*>(p.dx) + r * p.Cg;
      const float mean = p.cmean[r], rstd = p.crstd[r];
      float v[NV][V], d[NV][V], m1 = 0.0f, m2 = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) {
          read(x, i, v[i]);
          read(dy, i, d[i]);
        }
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) {
          float z[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            v[i][e] = (v[i][e] - mean) * rstd;
            z[e] = __builtin_fmaf(v[i][e], w[i][e], b[i][e]);
          }
          act_bwd<V>(p.act, z, d[i]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            dw[i][e] = __builtin_fmaf(d[i][e], v[i][e], dw[i][e]);
            db[i][e] += d[i][e];
            d[i][e] *= w[i][e];
            m1 += d[i][e];
            m2 = __builtin_fmaf(d[i][e], v[i][e], m2);
          }
        }
      m1 = team_sum<TL>(m1) * inv;
      m2 = team_sum<TL>(m2) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) {
#pragma unroll
          for (int e = 0; e < V; ++e) d[i][e] = rstd * (d[i][e] - m1 - v[i][e] * m2);
          write(dx, i, d[i]);
        }
    }
  }
  if (!p.dw) return;
  const bool join = TB % p.G == 0;                          // uniform: teams lt, lt + G, ... of the block share a group
  const int64_t row = join ? blockIdx.x : team / p.G;
  float* out = p.ws + row * 2 * p.C;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = g * p.Cg + (lane + TL * i) * V;
    if (join) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        red[0][e][threadIdx.x] = dw[i][e];
        red[1][e][threadIdx.x] = db[i][e];
      }
      __syncthreads();
      if (lt < p.G && (lane + TL * i) * V < p.Cg) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (RAG && e >= left(i)) break;
          float a = 0.0f, q = 0.0f;
          for (int k = lt; k < TB; k += p.G) {
            a += red[0][e][k * TL + lane];
            q += red[1][e][k * TL + lane];
          }
          out[c + e] = a;
          out[p.C + c + e] = q;
        }
      }
    } else if (in[i]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (RAG && e >= left(i)) break;
        out[c + e] = dw[i][e];
        out[p.C + c + e] = db[i][e];
      }
    }
  }
}

// d_weight, d_bias = sums over `rows` rows [2][C] of ws.  32 columns a block, 32 threads a column.
template <typename T>
__global__ __launch_bounds__(1024) void param_sum_kernel(const GnP p, const float* __restrict__ src, int64_t rows) {
  __shared__ float red[32][33];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + cl;          // column of [2 C]
  float a = 0.0f;
  if (c < 2 * (int64_t)p.C) {
    constexpr int U = 8;
    for (int64_t r = rl; r < rows; r += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = r + 32 * u < rows ? src[(r + 32 * u) * 2 * p.C + c] : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) a += v[u];
    }
  }
  red[rl][cl] = a;
  __syncthreads();
  if (rl == 0 && c < 2 * (int64_t)p.C) {
    float s = 0.0f;
    for (int k = 0; k < 32; ++k) s += red[k][cl];
    if (c < p.C) put_param<T>(p.dw, p.pdt, c, s);
    else put_param<T>(p.db, p.pdt, c - p.C, s);
  }
}

// ---- many pixels -------------------------------------------------------------------------------------------------------------------
// count, mean and centred sum of squares of two parts joined into the first
__device__ __forceinline__ void join_moments(float& n, float& m, float& s, float n2, float m2, float s2) {
  const float t = n + n2;
  if (n2 > 0.0f) {
    const float d = m2 - m, f = n2 / t;
    m = __builtin_fmaf(d, f, m);
    s += s2 + d * d * (n * f);
    n = t;
  }
}

// sample, part, pixels, first channel, its group, pixel lane and their number, channel vector of the block, vectors of a group in the
// block and this one's place among them
struct Place { int64_t n; int part; int64_t p0, p1; int c, g, row, rows, col, cgv, j; bool in; };

// Block -> (sample, part, channel slab), thread -> (channel vector, pixel lane).
template <int V> __device__ __forceinline__ Place place(const GnP& p) {
  Place q;
  const int slab = blockIdx.x % p.slabs, nv = p.Cg / V;
  const int64_t ns = blockIdx.x / p.slabs;
  const int split = (int)(ns % p.splits);
  q.n = ns / p.splits;
  q.p0 = split * (int64_t)p.chunk;
  q.p1 = min(p.L, q.p0 + p.chunk);
  q.rows = 256 / p.cvs;
  q.col = threadIdx.x % p.cvs;
  q.row = threadIdx.x / p.cvs;
  if (p.spg > 1) {
    const int piece = slab % p.spg;
    q.g = slab / p.spg;
    q.part = split * p.spg + piece;
    q.j = q.col;
    q.cgv = min(p.cvs, nv - piece * p.cvs);
    q.in = q.row < q.rows && q.col < q.cgv;
    q.c = q.g * p.Cg + (piece * p.cvs + q.col) * V;
  } else {
    q.part = split;
    q.c = (slab * p.cvs + q.col) * V;
    q.in = q.row < q.rows && q.c < p.C;
    q.g = q.c / p.Cg;
    q.cgv = nv;
    q.j = q.col % nv;
  }
  return q;
}

template <typename T, int V>
__global__ __launch_bounds__(256) void pixel_stats_kernel(const GnP p) {
  __shared__ float sn[256], sm[256], ss[256];
  const Place q = place<V>(p);
  const T* x = static_cast<const T*>(p.x) + q.n * p.L * p.C + q.c;
  float n = 0.0f, m = 0.0f, s = 0.0f;
  constexpr int U = V >= 4 ? 4 : 8;
  if (q.in) {
    for (int64_t r = q.p0 + q.row; r < q.p1; r += (int64_t)q.rows * U) {
      float v[U][V];
      float k = 0.0f, a = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + (int64_t)u * q.rows < q.p1) Vec<T, V>::load(x + (r + (int64_t)u * q.rows) * p.C, v[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + (int64_t)u * q.rows < q.p1) {
          k += V;
#pragma unroll
          for (int e = 0; e < V; ++e) a += v[u][e];
        }
      float mb = a / k, sb = 0.0f, d = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + (int64_t)u * q.rows < q.p1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float c = v[u][e] - mb;
            if constexpr (sizeof(T) == 4) d += c;
            sb = __builtin_fmaf(c, c, sb);
          }
        }
      if constexpr (sizeof(T) == 4) {
        d /= k;
        mb += d;
        sb = __builtin_fmaf(-d * k, d, sb);
        sb = sb < 0.0f ? 0.0f : sb;
      }
      join_moments(n, m, s, k, mb, sb);
    }
  }
  const int t = threadIdx.x;
  sn[t] = n; sm[t] = m; ss[t] = s;
  // pixel lanes, then the channel vectors of a group, halving each time
  for (int k = q.rows; k > 1;) {
    const int h = (k + 1) / 2;
    __syncthreads();
    if (q.row < k - h) {
      const int o = t + h * p.cvs;
      join_moments(n, m, s, sn[o], sm[o], ss[o]);
      sn[t] = n; sm[t] = m; ss[t] = s;
    }
    k = h;
  }
  for (int k = q.cgv; k > 1;) {
    const int h = (k + 1) / 2;
    __syncthreads();
    if (q.row == 0 && q.in && q.j < k - h) {
      join_moments(n, m, s, sn[t + h], sm[t + h], ss[t + h]);
      sn[t] = n; sm[t] = m; ss[t] = s;
    }
    k = h;
  }
  if (q.row == 0 && q.in && q.j == 0) {
    float* o = p.ws + ((q.n * p.splits * p.spg + q.part) * p.G + q.g) * 3;
    o[0] = n; o[1] = m; o[2] = s;
  }
}

// Where vectors reach over the border of a group: moments per channel and part -> ws [n][part][2][C] (mean, centred squares).
template <typename T, int V>
__global__ __launch_bounds__(256) void pixel_stats_mixed_kernel(const GnP p) {
  __shared__ float sn[256], sm[V][256], ss[V][256];
  const Place q = place<V>(p);
  const T* x = static_cast<const T*>(p.x) + q.n * p.L * p.C + q.c;
  float n = 0.0f, m[V], s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) m[e] = s[e] = 0.0f;
  constexpr int U = 8;
  if (q.in) {
    for (int64_t r = q.p0 + q.row; r < q.p1; r += (int64_t)q.rows * U) {
      float v[U][V], k = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + (int64_t)u * q.rows < q.p1) {
          Vec<T, V>::load(x + (r + (int64_t)u * q.rows) * p.C, v[u]);
          k += 1.0f;
        }
      const float ik = 1.0f / k, t = n + k, f = k / t, g = n * f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float a = 0.0f, b = 0.0f, o = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r + (int64_t)u * q.rows < q.p1) a += v[u][e];
        if (sizeof(T) == 4 || k == (float)U) a = rounded(a * ik);
        else a /= k;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r + (int64_t)u * q.rows < q.p1) {
            const float x = v[u][e] - a;
            if constexpr (sizeof(T) == 4) o += x;
            b = __builtin_fmaf(x, x, b);
          }
        if constexpr (sizeof(T) == 4) {
          const float h = o * ik;
          a += h;
          b = __builtin_fmaf(-h, o, b);
          b = b < 0.0f ? 0.0f : b;
        }
        const float d = a - m[e];
        m[e] = __builtin_fmaf(d, f, m[e]);
        s[e] += b + d * d * g;
      }
      n = t;
    }
  }
  const int t = threadIdx.x;
  sn[t] = n;
#pragma unroll
  for (int e = 0; e < V; ++e) { sm[e][t] = m[e]; ss[e][t] = s[e]; }
  for (int k = q.rows; k > 1;) {
    const int h = (k + 1) / 2;
    __syncthreads();
    if (q.row < k - h) {
      const int o = t + h * p.cvs;
      float n0 = n;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        n0 = n;
        join_moments(n0, m[e], s[e], sn[o], sm[e][o], ss[e][o]);
        sm[e][t] = m[e]; ss[e][t] = s[e];
      }
      n = n0;
      sn[t] = n;
    }
    k = h;
  }
  if (q.row == 0 && q.in) {
    float* o = p.ws + (q.n * p.splits + q.part) * 2 * p.C + q.c;
#pragma unroll
    for (int e = 0; e < V; ++e) { o[e] = m[e]; o[p.C + e] = s[e]; }
  }
}
// One block per (sample, group): the channels' moments of all parts joined -> mean, rstd.
__global__ __launch_bounds__(1024) void pixel_stats_join_kernel(const GnP p, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float sn[1024], sm[1024], ss[1024];
  const int64_t ng = blockIdx.x, sample = ng / p.G;
  const int g = (int)(ng % p.G), t = threadIdx.x;
  float n = 0.0f, m = 0.0f, s = 0.0f;
  for (int k = t; k < p.Cg * p.splits; k += blockDim.x) {
    const int part = k / p.Cg, c = g * p.Cg + k % p.Cg;
    const float* o = p.ws + (sample * p.splits + part) * 2 * p.C + c;
    join_moments(n, m, s, (float)min<int64_t>(p.chunk, p.L - (int64_t)part * p.chunk), o[0], o[p.C]);
  }
  sn[t] = n; sm[t] = m; ss[t] = s;
  for (int h = blockDim.x / 2; h >= 1; h >>= 1) {
    __syncthreads();
    if (t < h) {
      join_moments(n, m, s, sn[t + h], sm[t + h], ss[t + h]);
      sn[t] = n; sm[t] = m; ss[t] = s;
    }
  }
  if (t == 0) {
    const float r = 1.0f / sqrtf(s / n + p.eps);
    mean[ng] = m;
    rstd[ng] = r;
    if (p.mean) { p.mean[ng] = m; p.rstd[ng] = r; }
  }
}

template <typename T, int V, bool MIXED>
__global__ __launch_bounds__(256) void pixel_fwd_kernel(const GnP p) {
  __shared__ float sn[256], sm[256], ss[256];
  const Place q = place<V>(p);
  float mean[MIXED ? V : 1], rstd[MIXED ? V : 1];
  if constexpr (MIXED) {
    if (!q.in) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      mean[e] = p.cmean[q.n * p.G + (q.c + e) / p.Cg];
      rstd[e] = p.crstd[q.n * p.G + (q.c + e) / p.Cg];
    }
  } else {
  // the parts' moments of the block's groups: thread t joins parts t / groups, ... of group t % groups, then halves
  const int gpb = p.spg > 1 ? 1 : p.cvs / q.cgv, parts = p.splits * p.spg;
  const int g0 = p.spg > 1 ? q.g : (q.c - q.col * V) / p.Cg;
  const int t = threadIdx.x, gl = t % gpb, lanes = 256 / gpb, sl = t / gpb;
  float n = 0.0f, m = 0.0f, s = 0.0f;
  if (sl < lanes && g0 + gl < p.G)
    for (int k = sl; k < parts; k += lanes) {
      const float* o = p.ws + ((q.n * parts + k) * p.G + g0 + gl) * 3;
      join_moments(n, m, s, o[0], o[1], o[2]);
    }
  sn[t] = n; sm[t] = m; ss[t] = s;
  for (int k = min(lanes, parts); k > 1;) {
    const int h = (k + 1) / 2;
    __syncthreads();
    if (sl < k - h) {
      join_moments(n, m, s, sn[t + h * gpb], sm[t + h * gpb], ss[t + h * gpb]);
      sn[t] = n; sm[t] = m; ss[t] = s;
    }
    k = h;
  }
  __syncthreads();
  if (!q.in) return;
  const int mine = q.g - g0;
  mean[0] = sm[mine];
  rstd[0] = 1.0f / sqrtf(ss[mine] / sn[mine] + p.eps);
  if (p.mean && q.part == 0 && q.row == 0 && q.j == 0) {
    p.mean[q.n * p.G + q.g] = mean[0];
    p.rstd[q.n * p.G + q.g] = rstd[0];
  }
  }
  float w[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    w[e] = param<T>(p.w, p.pdt, q.c + e, 1.0f);
    b[e] = param<T>(p.b, p.pdt, q.c + e, 0.0f);
  }
  const T* x = static_cast<const T*>(p.x) + q.n * p.L * p.C + q.c;
  T* y = static_cast<T*>(p.y) + q.n * p.L * p.C + q.c;
  constexpr int U = 4;
  for (int64_t r = q.p0 + q.row; r < q.p1; r += (int64_t)q.rows * U) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + (int64_t)u * q.rows < q.p1) Vec<T, V>::load(x + (r + (int64_t)u * q.rows) * p.C, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + (int64_t)u * q.rows < q.p1) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] = __builtin_fmaf((v[u][e] - mean[MIXED ? e : 0]) * rstd[MIXED ? e : 0], w[e], b[e]);
        act_fwd<V>(p.act, v[u]);
        Vec<T, V>::store(y + (r + (int64_t)u * q.rows) * p.C, v[u]);
      }
  }
}

// per channel and part: sum dz xhat, sum dz  ->  ws [n][part][2][C]
template <typename T, int V, bool MIXED>
__global__ __launch_bounds__(256) void pixel_bwd_sums_kernel(const GnP p) {
  __shared__ float red[2][V][256];
  const Place q = place<V>(p);
  float dw[V], db[V];
#pragma unroll
  for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.0f;
  if (q.in) {
    float mean[MIXED ? V : 1], rstd[MIXED ? V : 1];
#pragma unroll
    for (int e = 0; e < (MIXED ? V : 1); ++e) {
      const int64_t ng = q.n * p.G + (MIXED ? (q.c + e) / p.Cg : q.g);
      mean[e] = p.cmean[ng];
      rstd[e] = p.crstd[ng];
    }
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[e] = param<T>(p.w, p.pdt, q.c + e, 1.0f);
      b[e] = param<T>(p.b, p.pdt, q.c + e, 0.0f);
    }
    const int64_t base = q.n * p.L * p.C + q.c;
    const T* x = static_cast<const T*>(p.x) + base;
    const T* dy = static_cast<const T*>(p.dy) + base;
    constexpr int U = 2;
    for (int64_t r = q.p0 + q.row; r < q.p1; r += (int64_t)q.rows * U) {
      float v[U][V], d[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + (int64_t)u * q.rows < q.p1) {
          Vec<T, V>::load(x + (r + (int64_t)u * q.rows) * p.C, v[u]);
          Vec<T, V>::load(dy + (r + (int64_t)u * q.rows) * p.C, d[u]);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + (int64_t)u * q.rows < q.p1) {
          float z[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            v[u][e] = (v[u][e] - mean[MIXED ? e : 0]) * rstd[MIXED ? e : 0];
            z[e] = __builtin_fmaf(v[u][e], w[e], b[e]);
          }
          act_bwd<V>(p.act, z, d[u]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            dw[e] = __builtin_fmaf(d[u][e], v[u][e], dw[e]);
            db[e] += d[u][e];
          }
        }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    red[0][e][threadIdx.x] = dw[e];
    red[1][e][threadIdx.x] = db[e];
  }
  __syncthreads();
  if (q.row == 0 && q.in) {
    float* out = p.ws + (q.n * p.splits + q.part / p.spg) * 2 * p.C + q.c;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float a = 0.0f, s = 0.0f;
      for (int k = 0; k < q.rows; ++k) {
        a += red[0][e][q.col + k * p.cvs];
        s += red[1][e][q.col + k * p.cvs];
      }
      out[e] = a;
      out[p.C + e] = s;
    }
  }
}

// One block per (sample, group): the parts' channel sums -> sums per channel [n][2][C] (for the parameters) and the group's two means.
template <typename T>
__global__ __launch_bounds__(256) void pixel_bwd_join_kernel(const GnP p, float* __restrict__ chan, float* __restrict__ coef) {
  __shared__ float red[2][256];
  const int64_t n = blockIdx.x / p.G;
  const int g = blockIdx.x % p.G, t = threadIdx.x;
  const int cc = min(p.Cg, 256), lanes = 256 / cc, cl = t % cc, sl = t / cc;   // channels at a time, threads of a channel
  float m1 = 0.0f, m2 = 0.0f;
  for (int cb = 0; cb < p.Cg; cb += cc) {
    const int c = g * p.Cg + cb + cl;
    const bool in = sl < lanes && cb + cl < p.Cg;
    float a = 0.0f, s = 0.0f;
    if (in) {
      const float* o = p.ws + n * p.splits * 2 * p.C + c;
      for (int k = sl; k < p.splits; k += lanes) {
        a += o[(int64_t)k * 2 * p.C];
        s += o[(int64_t)k * 2 * p.C + p.C];
      }
    }
    red[0][t] = a;
    red[1][t] = s;
    __syncthreads();
    if (in && sl == 0) {
      for (int k = 1; k < lanes; ++k) {
        a += red[0][t + k * cc];
        s += red[1][t + k * cc];
      }
      chan[n * 2 * p.C + c] = a;
      chan[n * 2 * p.C + p.C + c] = s;
      const float w = param<T>(p.w, p.pdt, c, 1.0f);
      m1 = __builtin_fmaf(w, s, m1);
      m2 = __builtin_fmaf(w, a, m2);
    }
    __syncthreads();
  }
  red[0][t] = m1;
  red[1][t] = m2;
  for (int h = 128; h >= 1; h >>= 1) {
    __syncthreads();
    if (t < h) {
      red[0][t] += red[0][t + h];
      red[1][t] += red[1][t + h];
    }
  }
  if (t == 0) {
    const float inv = 1.0f / ((float)p.L * (float)p.Cg);
    coef[blockIdx.x * 2] = red[0][0] * inv;
    coef[blockIdx.x * 2 + 1] = red[1][0] * inv;
  }
}

template <typename T, int V, bool MIXED>
__global__ __launch_bounds__(256) void pixel_bwd_dx_kernel(const GnP p, const float* __restrict__ coef) {
  const Place q = place<V>(p);
  if (!q.in) return;
  float mean[MIXED ? V : 1], rstd[MIXED ? V : 1], m1[MIXED ? V : 1], m2[MIXED ? V : 1];
#pragma unroll
  for (int e = 0; e < (MIXED ? V : 1); ++e) {
    const int64_t ng = q.n * p.G + (MIXED ? (q.c + e) / p.Cg : q.g);
    mean[e] = p.cmean[ng]; rstd[e] = p.crstd[ng];
    m1[e] = coef[2 * ng]; m2[e] = coef[2 * ng + 1];
  }
  float w[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    w[e] = param<T>(p.w, p.pdt, q.c + e, 1.0f);
    b[e] = param<T>(p.b, p.pdt, q.c + e, 0.0f);
  }
  const int64_t base = q.n * p.L * p.C + q.c;
  const T* x = static_cast<const T*>(p.x) + base;
  const T* dy = static_cast<const T*>(p.dy) + base;
  T* dx = static_cast<T*>(p.dx) + base;
  constexpr int U = 2;
  for (int64_t r = q.p0 + q.row; r < q.p1; r += (int64_t)q.rows * U) {
    float v[U][V], d[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + (int64_t)u * q.rows < q.p1) {
        Vec<T, V>::load(x + (r + (int64_t)u * q.rows) * p.C, v[u]);
        Vec<T, V>::load(dy + (r + (int64_t)u * q.rows) * p.C, d[u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + (int64_t)u * q.rows < q.p1) {
        float z[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[u][e] = (v[u][e] - mean[MIXED ? e : 0]) * rstd[MIXED ? e : 0];
          z[e] = __builtin_fmaf(v[u][e], w[e], b[e]);
        }
        act_bwd<V>(p.act, z, d[u]);
#pragma unroll
        for (int e = 0; e < V; ++e) d[u][e] = rstd[MIXED ? e : 0] * (d[u][e] * w[e] - m1[MIXED ? e : 0] - v[u][e] * m2[MIXED ? e : 0]);
        Vec<T, V>::store(dx + (r + (int64_t)u * q.rows) * p.C, d[u]);
      }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
struct Plan {
  int v;                       // elements of a vector
  bool tokens, mixed;          // mixed: rows of a token kernel are not whole vectors; vectors of a pixel kernel reach over groups
  int tl, nv, blocks, teams;   // tokens
  int64_t param_rows;          // rows [2][C] that param_sum adds
  int splits, chunk, cvs, slabs, spg;
};

int check(const mrl_group_norm* p, const char* what) {
  if (!p) MEM_FAIL(MRL_EINVAL, "%s: null description", what);
  if (p->dtype < MRL_F32 || p->dtype > MRL_F16) MEM_FAIL(MRL_EINVAL, "%s: dtype %d (float32, bfloat16 or float16)", what, p->dtype);
  if (p->param_dtype != p->dtype && p->param_dtype != MRL_F32) MEM_FAIL(MRL_EINVAL, "%s: weight and bias of the data's type or float32", what);
  if (p->act < MRL_ACT_NONE || p->act > MRL_ACT_GELU) MEM_FAIL(MRL_EINVAL, "%s: activation %d", what, p->act);
  if (p->batch < 0 || p->pixels < 0 || p->channels < 1) MEM_FAIL(MRL_EINVAL, "%s: batch %lld, pixels %lld, channels %d", what, (long long)p->batch, (long long)p->pixels, p->channels);
  if (p->groups < 1 || p->channels % p->groups) MEM_FAIL(MRL_EINVAL, "%s: %d channels are not %d groups", what, p->channels, p->groups);
  if (p->pixels > (int64_t(1) << 30) || p->channels > (1 << 24) || p->batch > (int64_t(1) << 30)) MEM_FAIL(MRL_EINVAL, "%s: sizes beyond 2^30", what);
  if (!(p->eps >= 0.0f)) MEM_FAIL(MRL_EINVAL, "%s: eps %g", what, p->eps);
  return MRL_OK;
}

Plan plan_of(const mrl_group_norm* p, bool backward) {
  Plan r{};
  const int cg = p->channels / p->groups, most_v = p->dtype == MRL_F32 ? 4 : 8;
  // Vectors of up to 16 bytes that divide a group.  Where that leaves single elements, the token kernels take 16-byte vectors and cut the
  // row's last one (with pairs that costs more than it gives: 38436 rows of 98 take 17.7 us so, 16.4 in pairs).  Where it leaves a
  // quarter of 16 bytes or less, the pixel kernels let a vector's channels belong to several groups, if the channels divide into wider
  // ones: 151 x 676 x 184 in 8 groups, fp16, both directions, 171 -> 107 us.
  r.v = most_v;
  while (cg % r.v) r.v /= 2;
  r.tokens = p->pixels == 1 && cdiv(cg, r.v == 1 && cg >= most_v ? most_v : r.v) <= 64 * 4;
  if (r.tokens && r.v == 1 && cg >= most_v) {
    r.mixed = true;
    r.v = most_v;
  } else if (!r.tokens && r.v * 4 <= most_v) {
    int all = most_v;
    while (p->channels % all) all /= 2;
    if (all > r.v) {
      r.mixed = true;
      r.v = all;
    }
  }
  const int nv = (int)cdiv(cg, r.v);
  if (r.tokens) {
    r.tl = 1;
    while (r.tl < nv && r.tl < 64) r.tl *= 2;
    r.nv = nv <= r.tl ? 1 : nv <= 2 * r.tl ? 2 : 4;
    const int tb = 256 / r.tl;
    const int64_t rows = p->batch * p->groups;
    // as many teams as fill the card (8 blocks a CU, 4 where the parameters' sums are kept), a whole number of groups
    const int64_t most = std::min<int64_t>(rows, (int64_t)(backward ? 1024 : 2048) * tb);
    int64_t teams = std::max<int64_t>(most / p->groups, 1) * p->groups;
    r.blocks = (int)cdiv(teams, tb);
    if (backward && tb % p->groups == 0) teams = (int64_t)r.blocks * tb;   // whole blocks: one row of sums each
    r.teams = (int)teams;
    r.param_rows = tb % p->groups == 0 ? r.blocks : teams / p->groups;
    return r;
  }
  // a block takes whole groups; a group of over 256 vectors is cut, and its pieces are joined like parts of the pixels
  r.spg = r.mixed ? 1 : (int)cdiv(nv, 256);
  r.cvs = r.mixed ? std::min(256, p->channels / r.v) : r.spg > 1 ? 256 : nv * std::max(1, std::min<int>(p->groups, 256 / nv));
  r.slabs = r.spg > 1 ? p->groups * r.spg : (int)cdiv(p->channels / r.v, r.cvs);
  const int64_t units = std::max<int64_t>(1, p->batch * r.slabs);
  // about 2048 blocks, and at least eight vectors for each thread
  int64_t splits = cdiv(2048, units);
  const int rows = 256 / r.cvs;
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, p->pixels / ((int64_t)rows * 8)));
  r.chunk = (int)std::max<int64_t>(1, cdiv(p->pixels, splits));
  r.splits = (int)std::max<int64_t>(1, cdiv(p->pixels, r.chunk));
  r.param_rows = p->batch;
  return r;
}

int64_t part_floats(const mrl_group_norm* p, const Plan& r, bool backward) {
  if (r.tokens) return backward ? r.param_rows * 2 * p->channels : 0;
  return p->batch * r.splits * (backward || r.mixed ? 2 * (int64_t)p->channels : 3 * (int64_t)p->groups * r.spg);
}
int64_t ws_floats(const mrl_group_norm* p, const Plan& r, bool backward) {
  int64_t n = part_floats(p, r, backward);
  if (!backward && !r.tokens && r.mixed) n += p->batch * p->groups * 2;
  if (backward && !r.tokens) n += p->batch * 2 * (int64_t)p->channels + p->batch * p->groups * 2;
  return n;
}

int check_ws(const mrl_group_norm* p, const Plan& r, bool backward, void* ws, int64_t bytes, const char* what) {
  const int64_t need = ws_floats(p, r, backward) * 4;
  if (need > 0 && (!ws || bytes < need)) MEM_FAIL(MRL_ENOSPC, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes, (long long)need);
  if (need > 0 && ((uintptr_t)ws & 15)) MEM_FAIL(MRL_EINVAL, "%s: workspace is not aligned", what);
  return MRL_OK;
}

GnP params_of(const mrl_group_norm* p, const Plan& r, void* ws) {
  GnP a{};
  a.N = p->batch; a.L = p->pixels; a.C = p->channels; a.G = p->groups; a.Cg = p->channels / p->groups; a.act = p->act;
  a.pdt = p->param_dtype == MRL_F32; a.eps = p->eps; a.teams = r.teams; a.splits = r.splits; a.chunk = r.chunk; a.cvs = r.cvs; a.slabs = r.slabs; a.spg = r.spg;
  a.ws = static_cast<float*>(ws);
  return a;
}

template <typename F> void with_team(const Plan& r, F&& f) {
  auto nv = [&](auto tl) {
    constexpr int TL = decltype(tl)::value;
    if (TL < 64 || r.nv == 1) f(tl, std::integral_constant<int, 1>());
    else if constexpr (TL == 64) {
      if (r.nv == 2) f(tl, std::integral_constant<int, 2>());
      else f(tl, std::integral_constant<int, 4>());
    }
  };
  switch (r.tl) {
    case 1: nv(std::integral_constant<int, 1>()); break;
    case 2: nv(std::integral_constant<int, 2>()); break;
    case 4: nv(std::integral_constant<int, 4>()); break;
    case 8: nv(std::integral_constant<int, 8>()); break;
    case 16: nv(std::integral_constant<int, 16>()); break;
    case 32: nv(std::integral_constant<int, 32>()); break;
    default: nv(std::integral_constant<int, 64>()); break;
  }
}

template <typename F> void with_flag(bool v, F&& f) {
  if (v) f(std::true_type());
  else f(std::false_type());
}
// kernels whose vectors are cut or reach over groups have more than one element
template <typename T, int V> void forward(GnP a, const Plan& r, hipStream_t st, float* stats) {
  with_flag(r.mixed, [&](auto mixed) {
    constexpr bool M = decltype(mixed)::value && V > 1;
    if (r.tokens) {
      with_team(r, [&](auto tl, auto nv) {
        hipLaunchKernelGGL((token_fwd_kernel<T, V, decltype(tl)::value, decltype(nv)::value, M>), dim3(r.blocks), dim3(256), 0, st, a);
      });
      return;
    }
    const dim3 grid((unsigned)(a.N * r.splits * r.slabs));
    if constexpr (M) {
      hipLaunchKernelGGL((pixel_stats_mixed_kernel<T, V>), grid, dim3(256), 0, st, a);
      const unsigned threads = a.Cg * a.splits > 4096 && a.N * a.G <= 65536 ? 1024 : 256;     // 5120 moments a group: 10 us, 26 by 256 threads; 184: 8 and 5 us
      hipLaunchKernelGGL(pixel_stats_join_kernel, dim3((unsigned)(a.N * a.G)), dim3(threads), 0, st, a, stats, stats + a.N * a.G);
      a.cmean = stats;
      a.crstd = stats + a.N * a.G;
    } else hipLaunchKernelGGL((pixel_stats_kernel<T, V>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((pixel_fwd_kernel<T, V, M>), grid, dim3(256), 0, st, a);
  });
}
template <typename T, int V> void backward(const GnP& a, const Plan& r, hipStream_t st, float* chan, float* coef) {
  const float* rows = a.ws;
  with_flag(r.mixed, [&](auto mixed) {
    constexpr bool M = decltype(mixed)::value && V > 1;
    if (r.tokens) {
      with_team(r, [&](auto tl, auto nv) {
        hipLaunchKernelGGL((token_bwd_kernel<T, V, decltype(tl)::value, decltype(nv)::value, M>), dim3(r.blocks), dim3(256), 0, st, a);
      });
      return;
    }
    const dim3 grid((unsigned)(a.N * r.splits * r.slabs));
    hipLaunchKernelGGL((pixel_bwd_sums_kernel<T, V, M>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((pixel_bwd_join_kernel<T>), dim3((unsigned)(a.N * a.G)), dim3(256), 0, st, a, chan, coef);
    hipLaunchKernelGGL((pixel_bwd_dx_kernel<T, V, M>), grid, dim3(256), 0, st, a, coef);
    rows = chan;
  });
  if (a.dw) hipLaunchKernelGGL((param_sum_kernel<T>), dim3((unsigned)cdiv(2 * (int64_t)a.C, 32)), dim3(1024), 0, st, a, rows, r.param_rows);
}

template <typename F> void with_type(int dtype, int v, F&& f) {
  auto by_v = [&](auto tag) {
    typedef decltype(tag) T;
    if constexpr (sizeof(T) == 2) {
      if (v == 8) return f(tag, std::integral_constant<int, 8>());
    }
    if (v == 4) return f(tag, std::integral_constant<int, 4>());
    if (v == 2) return f(tag, std::integral_constant<int, 2>());
    return f(tag, std::integral_constant<int, 1>());
  };
  if (dtype == MRL_F32) by_v(0.0f);
  else if (dtype == MRL_BF16) by_v((__bf16)0.0f);
  else by_v((_Float16)0.0f);
}

int check_grid(const mrl_group_norm* p, const Plan& r, const char* what) {
  // blocks of 256 threads, and a grid has less than 2^32 of them
  if (!r.tokens && (p->batch * r.splits * r.slabs >= (int64_t(1) << 24) || p->batch * p->groups >= (int64_t(1) << 24)))
    MEM_FAIL(MRL_EINVAL, "%s: %lld samples of %d groups (below 2^24 together)", what, (long long)p->batch, p->groups);
  return MRL_OK;
}

// Whole vectors lie on their own size: data on other addresses are refused.
int vec_of(const Plan& r, int dtype, std::initializer_list<const void*> ps) {
  const int es = dtype == MRL_F32 ? 4 : 2;
  const int n = r.tokens && r.mixed ? 1 : r.v;              // cut rows lie on any address anyway
  for (const void* q : ps)
    if ((uintptr_t)q % (uintptr_t)(n * es)) return 0;
  return 1;
}

}  // namespace

extern "C" int64_t mrl_group_norm_act_workspace_bytes(const mrl_group_norm* p, int32_t backward) {
  const int rc = check(p, "mrl_group_norm_act_workspace_bytes");
  if (rc) return rc;
  return ws_floats(p, plan_of(p, backward != 0), backward != 0) * 4;
}

extern "C" int mrl_group_norm_act(const mrl_group_norm* p, const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const char* what = "mrl_group_norm_act";
  int rc = check(p, what);
  if (rc) return rc;
  if (p->batch == 0 || p->pixels == 0) return MRL_OK;
  if (!x || !y) MEM_FAIL(MRL_EINVAL, "%s: null data", what);
  if (!mean != !rstd) MEM_FAIL(MRL_EINVAL, "%s: mean and rstd come together", what);
  const Plan r = plan_of(p, false);
  if ((rc = check_grid(p, r, what)) || (rc = check_ws(p, r, false, workspace, workspace_bytes, what))) return rc;
  if (!vec_of(r, p->dtype, {x, y})) MEM_FAIL(MRL_EINVAL, "%s: x and y have to be aligned to %d elements", what, r.v);
  GnP a = params_of(p, r, workspace);
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  hipStream_t st = static_cast<hipStream_t>(stream);
  with_type(p->dtype, r.v, [&](auto tag, auto v) { forward<decltype(tag), decltype(v)::value>(a, r, st, a.ws + part_floats(p, r, false)); });
  MEM_CHECK_LAUNCH(what);
  return MRL_OK;
}

extern "C" int mrl_group_norm_act_backward(const mrl_group_norm* p, const void* x, const void* dy, const void* weight, const void* bias, const float* mean,
                                           const float* rstd, void* dx, void* d_weight, void* d_bias, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "mrl_group_norm_act_backward";
  int rc = check(p, what);
  if (rc) return rc;
  if (!d_weight != !d_bias) MEM_FAIL(MRL_EINVAL, "%s: d_weight and d_bias come together", what);
  if (p->batch == 0 || p->pixels == 0) {
    if (d_weight) MEM_FAIL(MRL_EINVAL, "%s: no data to sum over", what);
    return MRL_OK;
  }
  if (!x || !dy || !dx || !mean || !rstd) MEM_FAIL(MRL_EINVAL, "%s: null data", what);
  const Plan r = plan_of(p, true);
  if ((rc = check_grid(p, r, what)) || (rc = check_ws(p, r, true, workspace, workspace_bytes, what))) return rc;
  if (!vec_of(r, p->dtype, {x, dy, dx})) MEM_FAIL(MRL_EINVAL, "%s: x, dy and dx have to be aligned to %d elements", what, r.v);
  GnP a = params_of(p, r, workspace);
  a.x = x; a.dy = dy; a.w = weight; a.b = bias; a.cmean = mean; a.crstd = rstd; a.dx = dx; a.dw = d_weight; a.db = d_bias;
  float* chan = a.ws + part_floats(p, r, true);
  float* coef = chan + p->batch * 2 * (int64_t)p->channels;
  hipStream_t st = static_cast<hipStream_t>(stream);
  with_type(p->dtype, r.v, [&](auto tag, auto v) { backward<decltype(tag), decltype(v)::value>(a, r, st, chan, coef); });
  MEM_CHECK_LAUNCH(what);
  return MRL_OK;
}
