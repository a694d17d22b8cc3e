// Layer norm, forward and backward, with the modulation a DiT block applies.
//
// Forward, per row of C channels:
//   mu = sum(x) / C,  rstd = 1 / sqrt(sum((x - mu)^2) / C + eps)
//   y  = (x - mu) * rstd * w + b,    w = weight (+ 1 when one_plus)
// Backward, with xh = (x - mu) * rstd and g = dy * w:
//   dx = rstd * (g - sum(g) / C - xh * sum(g * xh) / C)
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
// weight and bias are [G, C]: row r uses row r / (rows / G), so one launch
// normalises and modulates every frame or video of a batch.
//
// Both passes are bound by HBM: forward reads x and writes y, backward reads
// x and dy and writes dx.  A row stays in registers between the statistics
// and the result (mean first, then the centred squares: no cancellation), so
// each tensor crosses HBM once.  All sums are fp32.
//
// dw / db: a CTA owns a contiguous range of a group's rows and every column
// (thread = fixed columns), keeps its column sums in registers over its rows
// and writes them to a [parts, 2, C] workspace once; a second kernel adds the
// parts in order.  No atomics: the result does not depend on timing.
#include "pkv_f2.cuh"
#include "pkv_vec.cuh"

namespace pkv {
namespace {

constexpr int kNormThreads = 256;
constexpr int64_t kMaxCols = int64_t(1) << 20;

struct NormArgs {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* mean;
  float* rstd;
  int64_t x_rs, y_rs, rows, rows_per_group;
  int C, parts;  // parts: blocks of a group (norm_cols_fwd_kernel)
  float eps, plus;
};

// s / c, c = 1 / inv: for fp32 rows one step of Newton's method takes the product's
// rounding out, m + (s - m c) / c; 16-bit rows would not show it, and 37440 of 1536
// take 36 us without and 42 with it.
template <typename T>
__device__ __forceinline__ float mean_of(float s, float c, float inv) {
  const float m = s * inv;
  if (sizeof(T) == 2) return m;
  const float fixed = fmaf(fmaf(-m, c, s), inv, m);
  return fabsf(m) < INFINITY ? fixed : m;
}

// 1 / sqrt(v), v > 0: the approximation of 2 units in the last place, with one step
// of Newton's method for fp32 rows, y + y (1 - v y y) / 2.
template <typename T>
__device__ __forceinline__ float rstd_of(float v) {
  const float y = rsqrtf(v);
  if (sizeof(T) == 2) return y;
  const float fixed = fmaf(0.5f * y, fmaf(-v * y, y, 1.0f), y);
  return y > 0.0f && y < INFINITY ? fixed : y;
}

// Sum over the threads of a block (whole warps), the same in every thread.
// `red` holds 32 floats and is free again after the next barrier.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < nw; ++i) s += red[i];
  return s;
}

// Sums of N = 2 or 4 values over a block, the same in every thread, with one
// barrier.  A warp folds its values into one another on the way down the
// butterfly (6 shuffles for 4 values), lanes 0, 8, 16, 24 are left with one
// sum each.  `buf` ([warps][4]) must not be in use by an earlier call that a
// slower warp still reads: callers alternate two.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*buf)[4]) {
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  constexpr uint32_t kAll = 0xffffffffu;
  static_assert(N == 2 || N == 4);
  const bool up8 = lane & 8;
  float r;
  if constexpr (N == 4) {
    const bool up = lane & 16;
    float a0 = up ? v[2] : v[0], a1 = up ? v[3] : v[1];
    a0 += __shfl_xor_sync(kAll, up ? v[0] : v[2], 16);
    a1 += __shfl_xor_sync(kAll, up ? v[1] : v[3], 16);
    r = (up8 ? a1 : a0) + __shfl_xor_sync(kAll, up8 ? a0 : a1, 8);
  } else {
    r = (up8 ? v[1] : v[0]) + __shfl_xor_sync(kAll, up8 ? v[0] : v[1], 8);
    r += __shfl_xor_sync(kAll, r, 16);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) r += __shfl_xor_sync(kAll, r, o);
  if ((lane & 7) == 0) buf[threadIdx.x >> 5][lane >> 3] = r;
  __syncthreads();
  // lane 4 w + i adds value i of warps w, w + 8, ...; then across the lanes
  const int w0 = lane >> 2;
  r = w0 < nw ? buf[w0][lane & 3] : 0.0f;
  for (int w = w0 + 8; w < nw; w += 8) r += buf[w][lane & 3];
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) r += __shfl_xor_sync(kAll, r, o);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(kAll, r, i);
}

// E elements of a row's vectors as pairs (the last one padded with 0).
template <int E>
struct Pairs {
  static constexpr int kN = (E + 1) / 2;
  f2 p[kN];
};
template <typename T, int V, int NV>
__device__ __forceinline__ Pairs<V * NV> to_pairs(const Vec<T, V> (&v)[NV]) {
  Pairs<V * NV> r;
  float f[2 * r.kN];
  f[2 * r.kN - 1] = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) widen<T, V>(v[i], f + i * V);
#pragma unroll
  for (int i = 0; i < r.kN; ++i) r.p[i] = mk2(f[2 * i], f[2 * i + 1]);
  return r;
}
template <typename T, int V, int NV>
__device__ __forceinline__ void from_pairs(const Pairs<V * NV>& r, Vec<T, V> (&v)[NV]) {
  float f[2 * r.kN];
#pragma unroll
  for (int i = 0; i < r.kN; ++i) un2(r.p[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = narrow<T, V>(f + i * V);
}
__device__ __forceinline__ float fold(f2 a) {
  float lo, hi;
  un2(a, lo, hi);
  return lo + hi;
}

// What a thread does with its vectors of a row once they are in f: centre,
// normalise, modulate, round, store.
template <typename TX, typename TW, int V, int NV>
__device__ __forceinline__ void norm_store(const NormArgs& a, int64_t row, int tid, int tpr,
                                           int nvec, const float (&f)[NV][V], float rstd) {
  const int64_t g = uint32_t(row) / uint32_t(a.rows_per_group);  // (rows < 2^31)
  const TW* w = a.w ? static_cast<const TW*>(a.w) + g * a.C : nullptr;
  const TW* b = a.b ? static_cast<const TW*>(a.b) + g * a.C : nullptr;
  TX* y = static_cast<TX*>(a.y) + row * a.y_rs;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = tid + i * tpr;
    if (j < nvec) {
      float r[V], t2[V];
#pragma unroll
      for (int e = 0; e < V; ++e) r[e] = f[i][e] * rstd;
      if (w) {
        ld_f32<TW, V>(w + j * V, t2);
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] *= t2[e] + a.plus;
      }
      if (b) {
        ld_f32<TW, V>(b + j * V, t2);
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] += t2[e];
      }
      st_vec<TX, V>(y + j * V, narrow<TX, V>(r));
    }
  }
}

// A block a row: V elements a vector, NV vectors a thread in registers.
template <typename TX, typename TW, int V, int NV>
__global__ void __launch_bounds__(1024) norm_fwd_kernel(NormArgs a) {
  __shared__ float red[2][32];
  const int tid = threadIdx.x, tpr = blockDim.x;
  const int64_t row = blockIdx.x;
  const int nvec = a.C / V;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_rs;
  float f[NV][V];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = tid + i * tpr;
    if (j < nvec) {
      widen<TX, V>(ld_vec<TX, V>(x + j * V), f[i]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[i][e] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) s += f[i][e];
  const float inv_c = 1.0f / float(a.C);
  const float mu = mean_of<TX>(block_sum(s, red[0]), float(a.C), inv_c);
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (tid + i * tpr < nvec)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[i][e] -= mu;
        q = fmaf(f[i][e], f[i][e], q);
      }
  const float rstd = rstd_of<TX>(mean_of<TX>(block_sum(q, red[1]), float(a.C), inv_c) + a.eps);
  if (tid == 0) {
    if (a.mean) a.mean[row] = mu;
    if (a.rstd) a.rstd[row] = rstd;
  }
  norm_store<TX, TW, V, NV>(a, row, tid, tpr, nvec, f, rstd);
}

// Short rows: L lanes a row, 32 / L rows a warp, one vector a lane; the next
// seven rounds' rows are on their way into shared memory while one is in
// registers, so HBM stays busy through the reductions.  Each lane copies exactly
// what it will read: no barriers.  200 000 rows of 64 bf16: 17 us, with a block
// a row 66.
constexpr int kShortStages = 8;

template <typename TX, typename TW, int V, int L>
__global__ void __launch_bounds__(kNormThreads) norm_short_kernel(NormArgs a) {
  __shared__ Vec<TX, V> ring[kShortStages][kNormThreads];
  constexpr int kPer = kNormThreads / L;  // rows of a block's round
  const int tid = threadIdx.x, lane = tid % L;
  const int64_t step = int64_t(gridDim.x) * kPer;
  const int64_t first = blockIdx.x * int64_t(kPer) + tid / L;
  const int nvec = a.C / V;
  const float inv_c = 1.0f / float(a.C);
  auto fetch = [&](int64_t row, int st) {
    if (row < a.rows && lane < nvec)
      cp_async<TX, V>(&ring[st][tid], static_cast<const TX*>(a.x) + row * a.x_rs + lane * V);
    cp_commit();  // an empty group counts too
  };
  for (int i = 0; i < kShortStages - 1; ++i) fetch(first + i * step, i);
  int st = 0;
  // (the whole warp goes on while one of its rows is there: shuffles)
  for (int64_t row = first; row - tid / L < a.rows; row += step) {
    cp_wait<kShortStages - 2>();
    const bool live = row < a.rows && lane < nvec;
    float f[1][V];
    if (live)
      widen<TX, V>(ring[st][tid], f[0]);
    else
#pragma unroll
      for (int e = 0; e < V; ++e) f[0][e] = 0.0f;
    // the slot read one round ago is free: its values are in registers
    fetch(row + (kShortStages - 1) * step, st == 0 ? kShortStages - 1 : st - 1);
    st = st + 1 == kShortStages ? 0 : st + 1;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) s += f[0][e];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mu = mean_of<TX>(s, float(a.C), inv_c);
    float q = 0.0f;
    if (lane < nvec)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[0][e] -= mu;
        q = fmaf(f[0][e], f[0][e], q);
      }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    const float rstd = rstd_of<TX>(mean_of<TX>(q, float(a.C), inv_c) + a.eps);
    if (row < a.rows) {
      if (lane == 0) {
        if (a.mean) a.mean[row] = mu;
        if (a.rstd) a.rstd[row] = rstd;
      }
      norm_store<TX, TW, V, 1>(a, row, lane, L, nvec, f, rstd);
    }
  }
}

// A block a range of a group's rows, every column (thread = fixed columns, as
// the backward pass): weight and bias are read once and stay in registers,
// R rows share the two barriers of their statistics, and the next
// rounds' rows are on their way into shared memory meanwhile.  37440 rows of
// 1536 bf16 take 36 us, 230 MB at 6.4 TB/s, the copy rate (one launch behind an L2
// flush; 43 in a steady loop); a warp a row, loading the weights for every row,
// took 62.
// (16-bit single elements are too small for asynchronous copies: loaded
// directly.)
constexpr int kColStages = 3;
__host__ __device__ constexpr int fwd_rows(int elems) { return elems <= 8 ? 4 : 2; }

template <typename TX, typename TW, int V, int NV, int kThreads>
__global__ void __launch_bounds__(kThreads, V * NV <= 8 ? 768 / kThreads : 1)
    norm_cols_fwd_kernel(NormArgs a) {
  constexpr int E = V * NV, R = fwd_rows(E);
  constexpr bool kRing = V * sizeof(TX) >= 4;
  __shared__ __align__(16) float red[2][kThreads / 32][4];
  extern __shared__ __align__(16) uint8_t raw[];
  const int tid = threadIdx.x, nthr = blockDim.x;
  Vec<TX, V>* ring = reinterpret_cast<Vec<TX, V>*>(raw) + tid;  // [stage][row][NV][nthr]
  const int64_t grp = blockIdx.x / a.parts;
  const int p = int(blockIdx.x - grp * a.parts);
  const int64_t r0 = grp * a.rows_per_group + a.rows_per_group * p / a.parts;
  const int64_t r1 = grp * a.rows_per_group + a.rows_per_group * (p + 1) / a.parts;
  const int nvec = a.C / V;
  const float inv_c = 1.0f / float(a.C);
  const int n = int(r1 - r0);  // rows of this block
  const TX* xp = static_cast<const TX*>(a.x) + r0 * a.x_rs + tid * V;
  TX* yp = static_cast<TX*>(a.y) + r0 * a.y_rs + tid * V;
  int ahead = 0;  // rows asked for
  auto fetch = [&](int st) {
    if constexpr (kRing) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (ahead + k < n)
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (tid + i * nthr < nvec)
              cp_async<TX, V>(ring + ((st * R + k) * NV + i) * nthr, xp + i * nthr * V);
        xp += a.x_rs;
      }
      ahead += R;
      cp_commit();
    }
  };
  for (int i = 0; i < kColStages - 1; ++i) fetch(i);
  Pairs<E> w, b;
  {
    const TW* wp = a.w ? static_cast<const TW*>(a.w) + grp * a.C : nullptr;
    const TW* bp = a.b ? static_cast<const TW*>(a.b) + grp * a.C : nullptr;
    float fw[E], fb[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = tid + i * nthr;
      float tw[V], tb[V];
      if (wp && j < nvec) ld_f32<TW, V>(wp + j * V, tw);
      if (bp && j < nvec) ld_f32<TW, V>(bp + j * V, tb);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        fw[i * V + e] = wp && j < nvec ? tw[e] + a.plus : 1.0f;
        fb[i * V + e] = bp && j < nvec ? tb[e] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < w.kN; ++i) {
      w.p[i] = mk2(fw[2 * i], 2 * i + 1 < E ? fw[(2 * i + 1) % E] : 0.0f);
      b.p[i] = mk2(fb[2 * i], 2 * i + 1 < E ? fb[(2 * i + 1) % E] : 0.0f);
    }
  }
  int st = 0;
  for (int r = 0; r < n; r += R) {
    if constexpr (kRing) cp_wait<kColStages - 2>();
    Pairs<E> f[R];
    float s[R];
    Vec<TX, V> direct[kRing ? 1 : R][NV];
    if constexpr (!kRing) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (r + k < n && tid + i * nthr < nvec)
            direct[k][i] = ld_vec<TX, V>(xp + i * nthr * V);
        xp += a.x_rs;
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      Vec<TX, V> v[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (r + k < n && tid + i * nthr < nvec) {
          if constexpr (kRing)
            v[i] = ring[((st * R + k) * NV + i) * nthr];
          else
            v[i] = direct[k][i];
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[i].v[e] = from_f32<TX>(0.0f);
        }
      }
      f[k] = to_pairs<TX, V, NV>(v);
      f2 t = f[k].p[0];
#pragma unroll
      for (int i = 1; i < f[k].kN; ++i) t = add2(t, f[k].p[i]);
      s[k] = fold(t);
    }
    fetch(st == 0 ? kColStages - 1 : st - 1);
    st = st + 1 == kColStages ? 0 : st + 1;
    block_sums<R>(s, red[0]);
    float mu[R], q[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      mu[k] = mean_of<TX>(s[k], float(a.C), inv_c);
      const f2 m2 = mk2(mu[k], mu[k]);
      f2 t = mk2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < f[k].kN; ++i) f[k].p[i] = sub2(f[k].p[i], m2);
      // columns that are not there hold -mu now: leave them out
#pragma unroll
      for (int i = 0; i < f[k].kN; ++i) {
        const int e0 = 2 * i, e1 = 2 * i + 1;
        const bool in0 = tid + e0 / V * nthr < nvec;
        const bool in1 = e1 < E && tid + e1 % E / V * nthr < nvec;
        if (in0 && in1) {
          t = fma2(f[k].p[i], f[k].p[i], t);
        } else if (in0) {
          float lo, hi, tl, th;
          un2(f[k].p[i], lo, hi);
          un2(t, tl, th);
          t = mk2(fmaf(lo, lo, tl), th);
        }
      }
      q[k] = fold(t);
    }
    block_sums<R>(q, red[1]);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (r + k >= n) break;
      const float rstd = rstd_of<TX>(mean_of<TX>(q[k], float(a.C), inv_c) + a.eps);
      if (tid == 0 && a.mean) a.mean[r0 + r + k] = mu[k];
      if (tid == 0 && a.rstd) a.rstd[r0 + r + k] = rstd;
      const f2 r2 = mk2(rstd, rstd);
#pragma unroll
      for (int i = 0; i < f[k].kN; ++i) f[k].p[i] = fma2(mul2(f[k].p[i], r2), w.p[i], b.p[i]);
      Vec<TX, V> v[NV];
      from_pairs<TX, V, NV>(f[k], v);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * nthr < nvec) st_vec<TX, V>(yp + i * nthr * V, v[i]);
      yp += a.y_rs;
    }
  }
}

// Rows too long for registers: the row is read three times, from L2 after the
// first.
template <typename TX, typename TW>
__global__ void __launch_bounds__(1024) norm_fwd_long_kernel(NormArgs a) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_rs;
  float s = 0.0f;
  for (int j = threadIdx.x; j < a.C; j += blockDim.x) s += to_f32(x[j]);
  const float mu = block_sum(s, red[0]) / float(a.C);
  float q = 0.0f;
  for (int j = threadIdx.x; j < a.C; j += blockDim.x) {
    const float d = to_f32(x[j]) - mu;
    q = fmaf(d, d, q);
  }
  const float rstd = rstd_of<TX>(block_sum(q, red[1]) / float(a.C) + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mu;
    if (a.rstd) a.rstd[row] = rstd;
  }
  const int64_t g = row / a.rows_per_group;
  const TW* w = a.w ? static_cast<const TW*>(a.w) + g * a.C : nullptr;
  const TW* b = a.b ? static_cast<const TW*>(a.b) + g * a.C : nullptr;
  TX* y = static_cast<TX*>(a.y) + row * a.y_rs;
  for (int j = threadIdx.x; j < a.C; j += blockDim.x) {
    float r = (to_f32(x[j]) - mu) * rstd;
    if (w) r *= to_f32(w[j]) + a.plus;
    if (b) r += to_f32(b[j]);
    y[j] = from_f32<TX>(r);
  }
}

struct NormBwdArgs {
  const void* dy;
  const void* x;
  const void* w;
  const float* mean;
  const float* rstd;
  void* dx;
  float* part;  // [groups * parts][2][C] column sums, or nullptr
  void* dw;     // the sums themselves where a group is one part, or nullptr
  void* db;
  int64_t dy_rs, x_rs, dx_rs, rows_per_group;
  int C, parts;
  float plus;
};

// Rows of one reduction round, and rounds of x and dy on their way into
// shared memory.
__host__ __device__ constexpr int bwd_stages(int stage_bytes) { return stage_bytes < 128 ? 4 : 3; }
__host__ __device__ constexpr int bwd_rows(int elems) { return elems <= 8 ? 2 : 1; }

// CTA (group, part): its rows, every column; V * NV columns a thread.  37440 rows
// of 1536 bf16 take 64 us, 345 MB at 5.4 TB/s (70 in a steady loop, with the sum of
// the parts): about 1000 warp instructions a row keep the issue slots 56% busy.  Rows loaded when needed 154 us, the same
// through shared memory ahead of use 102, conversions in pairs 82; the rest came
// from a grid of one wave (448 blocks on 444 places had cost a second one).
// 16-bit single elements (V = 1) are too small for asynchronous copies and
// are loaded directly.
template <typename TX, typename TW, int V, int NV, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads <= 192 ? 3 : kThreads <= 256 && V * NV <= 8 ? 2 : 1)
    norm_bwd_kernel(NormBwdArgs a) {
  constexpr int R = bwd_rows(V * NV), E = V * NV;
  constexpr bool kRing = V * sizeof(TX) >= 4;
  constexpr int kStages = bwd_stages(R * 2 * NV * V * sizeof(TX));
  __shared__ __align__(16) float red[2][kThreads / 32][4];
  extern __shared__ __align__(16) uint8_t raw[];
  const int tid = threadIdx.x, nthr = blockDim.x;
  Vec<TX, V>* ring = reinterpret_cast<Vec<TX, V>*>(raw) + tid;  // [stage][row][x, dy][NV][nthr]
  const int64_t grp = blockIdx.x / a.parts;
  const int p = int(blockIdx.x - grp * a.parts);
  const int64_t r0 = grp * a.rows_per_group + a.rows_per_group * p / a.parts;
  const int64_t r1 = grp * a.rows_per_group + a.rows_per_group * (p + 1) / a.parts;
  const int nvec = a.C / V;
  const float inv_c = 1.0f / float(a.C);
  const TW* wp = a.w ? static_cast<const TW*>(a.w) + grp * a.C : nullptr;
  const int n = int(r1 - r0);  // rows of this block
  const TX* xp = static_cast<const TX*>(a.x) + r0 * a.x_rs + tid * V;
  const TX* dp = static_cast<const TX*>(a.dy) + r0 * a.dy_rs + tid * V;
  TX* op = static_cast<TX*>(a.dx) + r0 * a.dx_rs + tid * V;
  int ahead = 0;  // rows asked for
  auto fetch = [&](int st) {
    if constexpr (kRing) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (ahead + k < n)
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (tid + i * nthr < nvec) {
              Vec<TX, V>* slot = ring + (((st * R + k) * 2) * NV + i) * nthr;
              cp_async<TX, V>(slot, xp + i * nthr * V);
              cp_async<TX, V>(slot + NV * nthr, dp + i * nthr * V);
            }
        xp += a.x_rs;
        dp += a.dy_rs;
      }
      ahead += R;
      cp_commit();
    }
  };
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  Pairs<E> w, aw, ab;
  {
    float fw[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = tid + i * nthr;
      float tw[V];
      if (wp && j < nvec) ld_f32<TW, V>(wp + j * V, tw);
#pragma unroll
      for (int e = 0; e < V; ++e) fw[i * V + e] = wp && j < nvec ? tw[e] + a.plus : 1.0f;
    }
#pragma unroll
    for (int i = 0; i < w.kN; ++i) {
      w.p[i] = mk2(fw[2 * i], 2 * i + 1 < E ? fw[(2 * i + 1) % E] : 0.0f);
      aw.p[i] = ab.p[i] = mk2(0.0f, 0.0f);
    }
  }
  int round = 0, st = 0;
  for (int r = 0; r < n; r += R, ++round) {
    Pairs<E> xh[R], gr[R];
    float rs[R], c[2 * R];
    if constexpr (kRing) cp_wait<kStages - 2>();
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const bool live = r + k < n;
      const float mu = live ? a.mean[r0 + r + k] : 0.0f;
      rs[k] = live ? a.rstd[r0 + r + k] : 0.0f;
      Vec<TX, V> vx[NV], vd[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (live && tid + i * nthr < nvec) {
          if constexpr (kRing) {
            const Vec<TX, V>* slot = ring + (((st * R + k) * 2) * NV + i) * nthr;
            vx[i] = slot[0];
            vd[i] = slot[NV * nthr];
          } else {
            vx[i] = ld_vec<TX, V>(xp + i * nthr * V);
            vd[i] = ld_vec<TX, V>(dp + i * nthr * V);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) vx[i].v[e] = vd[i].v[e] = from_f32<TX>(0.0f);
        }
      }
      if constexpr (!kRing) {
        xp += a.x_rs;
        dp += a.dy_rs;
      }
      // (columns and rows that are not there have dy = 0; such rows rstd = 0)
      xh[k] = to_pairs<TX, V, NV>(vx);
      gr[k] = to_pairs<TX, V, NV>(vd);
      const f2 m2 = mk2(mu, mu), r2 = mk2(rs[k], rs[k]);
      f2 s1 = mk2(0.0f, 0.0f), s2 = s1;
#pragma unroll
      for (int i = 0; i < w.kN; ++i) {
        const f2 d = gr[k].p[i];
        xh[k].p[i] = mul2(sub2(xh[k].p[i], m2), r2);
        gr[k].p[i] = mul2(d, w.p[i]);
        s1 = add2(s1, gr[k].p[i]);
        s2 = fma2(gr[k].p[i], xh[k].p[i], s2);
        aw.p[i] = fma2(d, xh[k].p[i], aw.p[i]);
        ab.p[i] = add2(ab.p[i], d);
      }
      c[2 * k] = fold(s1);
      c[2 * k + 1] = fold(s2);
    }
    // the slot read one round ago is free: its values were in registers
    fetch(st == 0 ? kStages - 1 : st - 1);
    st = st + 1 == kStages ? 0 : st + 1;
    // two buffers in turn: a warp may write the next round's while another
    // still reads this one's
    block_sums<2 * R>(c, red[round & 1]);
    if (a.dx != nullptr) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (r + k >= n) break;
        const float n1 = -mean_of<TX>(c[2 * k], float(a.C), inv_c);
        const float n2 = -mean_of<TX>(c[2 * k + 1], float(a.C), inv_c);
        const f2 c1 = mk2(n1, n1), c2 = mk2(n2, n2), r2 = mk2(rs[k], rs[k]);
#pragma unroll
        for (int i = 0; i < w.kN; ++i)
          gr[k].p[i] = mul2(fma2(xh[k].p[i], c2, add2(gr[k].p[i], c1)), r2);
        Vec<TX, V> v[NV];
        from_pairs<TX, V, NV>(gr[k], v);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (tid + i * nthr < nvec) st_vec<TX, V>(op + i * nthr * V, v[i]);
        op += a.dx_rs;
      }
    }
  }
  if (a.part != nullptr || a.dw != nullptr || a.db != nullptr) {
    float* pw = a.part + int64_t(blockIdx.x) * 2 * a.C;
    TW* dw = static_cast<TW*>(a.dw) + grp * a.C;
    TW* db = static_cast<TW*>(a.db) + grp * a.C;
    float sw[2 * w.kN], sb[2 * w.kN];
#pragma unroll
    for (int i = 0; i < w.kN; ++i) {
      un2(aw.p[i], sw[2 * i], sw[2 * i + 1]);
      un2(ab.p[i], sb[2 * i], sb[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = tid + i * nthr;
      if (j < nvec)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (a.part != nullptr) {
            pw[j * V + e] = sw[i * V + e];
            pw[a.C + j * V + e] = sb[i * V + e];
          } else {
            if (a.dw != nullptr) dw[j * V + e] = from_f32<TW>(sw[i * V + e]);
            if (a.db != nullptr) db[j * V + e] = from_f32<TW>(sb[i * V + e]);
          }
        }
    }
  }
}

// Rows too long for registers: dx by one CTA a row ...
template <typename TX, typename TW>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(NormBwdArgs a) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_rs;
  const TX* d = static_cast<const TX*>(a.dy) + row * a.dy_rs;
  TX* dx = static_cast<TX*>(a.dx) + row * a.dx_rs;
  const TW* w = a.w ? static_cast<const TW*>(a.w) + row / a.rows_per_group * a.C : nullptr;
  const float mu = a.mean[row], rs = a.rstd[row];
  float c1 = 0.0f, c2 = 0.0f;
  for (int j = threadIdx.x; j < a.C; j += blockDim.x) {
    const float g = to_f32(d[j]) * (w ? to_f32(w[j]) + a.plus : 1.0f);
    c1 += g;
    c2 = fmaf(g, (to_f32(x[j]) - mu) * rs, c2);
  }
  c1 = block_sum(c1, red[0]) / float(a.C);
  c2 = block_sum(c2, red[1]) / float(a.C);
  for (int j = threadIdx.x; j < a.C; j += blockDim.x) {
    const float g = to_f32(d[j]) * (w ? to_f32(w[j]) + a.plus : 1.0f);
    dx[j] = from_f32<TX>(rs * (g - c1 - (to_f32(x[j]) - mu) * rs * c2));
  }
}

// ... and the column sums by one thread a column of a (group, part).
template <typename TX>
__global__ void __launch_bounds__(kNormThreads) norm_cols_kernel(NormBwdArgs a) {
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  if (c >= a.C) return;
  const int64_t grp = blockIdx.x / a.parts;
  const int p = int(blockIdx.x - grp * a.parts);
  const int64_t r0 = grp * a.rows_per_group + a.rows_per_group * p / a.parts;
  const int64_t r1 = grp * a.rows_per_group + a.rows_per_group * (p + 1) / a.parts;
  float sw = 0.0f, sb = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float d = to_f32(static_cast<const TX*>(a.dy)[r * a.dy_rs + c]);
    const float xh = (to_f32(static_cast<const TX*>(a.x)[r * a.x_rs + c]) - a.mean[r]) * a.rstd[r];
    sw = fmaf(d, xh, sw);
    sb += d;
  }
  a.part[int64_t(blockIdx.x) * 2 * a.C + c] = sw;
  a.part[int64_t(blockIdx.x) * 2 * a.C + a.C + c] = sb;
}

// Column sums of a group's parts, in a fixed order, rounded to the weight's
// type: VC columns a thread, 32 threads x 8 slices of the parts a block, eight
// parts of a slice on their way at once; the slices meet in shared memory.
template <typename TW, int VC>
__global__ void __launch_bounds__(256)
    norm_parts_kernel(const float* part, int parts, int C, TW* dw, TW* db) {
  constexpr int kCols = 32 * VC, kMany = 8;
  __shared__ float sm[2][8][kCols];
  const int lane = threadIdx.x & 31, sl = threadIdx.x >> 5;
  const int c = blockIdx.y * kCols + lane * VC;
  const int64_t grp = blockIdx.x;
  float s[2][VC] = {};
  if (c < C) {
    const float* q = part + grp * parts * 2 * int64_t(C) + c;
    for (int p = sl; p < parts; p += 8 * kMany) {
      Vec<float, VC> v[kMany][2];
#pragma unroll
      for (int i = 0; i < kMany; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (p + 8 * i < parts) v[i][k] = ld_vec<float, VC>(q + (int64_t(p + 8 * i) * 2 + k) * C);
#pragma unroll
      for (int i = 0; i < kMany; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (p + 8 * i < parts)
#pragma unroll
            for (int e = 0; e < VC; ++e) s[k][e] += v[i][k].v[e];
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < VC; ++e) sm[k][sl][lane * VC + e] = s[k][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * kCols; i += 256) {
    const int k = i / kCols, col = i - k * kCols;
    TW* out = k ? db : dw;
    if (out == nullptr || blockIdx.y * kCols + col >= C) continue;
    float t = 0.0f;
#pragma unroll
    for (int x = 0; x < 8; ++x) t += sm[k][x][col];
    out[grp * C + blockIdx.y * kCols + col] = from_f32<TW>(t);
  }
}

// Blocks that share a group's rows: at most `per_sm` an SM over all groups (one
// more would be a second wave), at least `least` rows each.
int64_t row_parts(int64_t rows_per_group, int64_t groups, int per_sm, int least) {
  const int64_t want = int64_t(sm_count()) * per_sm / groups;
  const int64_t most = (rows_per_group + least - 1) / least;
  const int64_t p = want < most ? want : most;
  return p < 1 ? 1 : p;
}
// Backward: three blocks of 192 threads an SM (what the registers allow), more of the
// smaller ones that short rows (16-byte vectors) leave.  us with two thirds / this /
// four thirds of them, 60 M elements of bf16: 1536 columns 69.4 / 69.8 / 79.7, 1024
// 78.5 / 70.0 / 71.2, 64 columns 170 / 172 / 172; but 256 85.8 / 97.6 / 118.7 and 128
// 132 / 147 / 167, where fewer would do.
int64_t bwd_parts(int64_t rows_per_group, int64_t groups, int64_t cols) {
  const int64_t thr = (cols / 8 + 31) / 32 * 32;
  const int per_sm = thr >= 192 ? 3 : thr <= 32 ? 18 : int(576 / thr);
  return row_parts(rows_per_group, groups, per_sm, 4);
}

// A group of one part needs no second pass and no workspace (rows in registers
// only: every width up to 8192 is).
bool one_pass(int64_t parts, int64_t cols) { return parts == 1 && cols <= 8192; }

constexpr int round_warp(int n) { return (n + 31) / 32 * 32; }

template <typename TX, typename TW, int V, int L>
int short_fwd(const NormArgs& a, cudaStream_t s) {
  const int64_t need = (a.rows + kNormThreads / L - 1) / (kNormThreads / L);
  const int64_t most = int64_t(sm_count()) * 5;
  norm_short_kernel<TX, TW, V, L><<<int(need < most ? need : most), kNormThreads, 0, s>>>(a);
  return launch_status();
}

template <typename TX, typename TW, int V, int NV, int kThreads>
int cols_fwd(NormArgs a, cudaStream_t s) {
  const int thr = round_warp((a.C / V + NV - 1) / NV);
  constexpr int R = fwd_rows(V * NV);
  constexpr size_t per = V * sizeof(TX) >= 4 ? size_t(kColStages) * R * NV * V * sizeof(TX) : 0;
  static_assert(per * kThreads <= 200 * 1024, "the rounds of a block fit its shared memory");
  static std::mutex mu;
  static int done[kMaxDevices] = {};
  if (smem_opt_in(done, mu, norm_cols_fwd_kernel<TX, TW, V, NV, kThreads>, per * kThreads) <= 0) {
    cudaGetLastError();
    return PKV_ELAUNCH;
  }
  const int64_t groups = a.rows / a.rows_per_group;
  const int per_sm = V * NV <= 8 ? 768 / thr : 1;  // (what the registers allow)
  a.parts = int(row_parts(a.rows_per_group, groups, per_sm > 0 ? per_sm : 1, 2 * R));
  const int64_t grid = groups * a.parts;
  if (grid >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  norm_cols_fwd_kernel<TX, TW, V, NV, kThreads><<<int(grid), thr, per * thr, s>>>(a);
  return launch_status();
}

template <typename TX, typename TW, int V>
int launch_fwd(const NormArgs& a, cudaStream_t s) {
  const int nvec = a.C / V;
  if (a.rows >= int64_t(sm_count()) * 16) {
    // rows enough to fill the GPU.  Short ones: a few lanes a row; longer
    // ones, in groups that give a block rows to share its weights over: fixed
    // columns.  us, a block a row / these forms, at 8, 16 and 64 rows an SM: 256 bf16
    // 2.5 / 2.3, 3.0 / 2.5, 6.7 / 4.8; 1536 bf16 4.0 / 4.1, 6.2 / 4.8, 18.9 / 10.4;
    // 520 fp32 3.3 / 3.9, 5.0 / 4.3, 13.8 / 8.2; 1535 bf16 8.3 / 10.0, 12.0 / 11.3,
    // 39 / 29.  Rows of 8 KB and odd fp32 ones gain nothing from them: 4096 bf16
    // 5.9 / 6.4, 9.8 / 10.4, 35.2 / 36.0; 1111 fp32 5.4 / 8.9, 9.1 / 9.9, 29.5 / 35.9.
    if constexpr (V * sizeof(TX) >= 4) {
      if (nvec <= 4) return short_fwd<TX, TW, V, 4>(a, s);
      if (nvec <= 8) return short_fwd<TX, TW, V, 8>(a, s);
      if (nvec <= 16) return short_fwd<TX, TW, V, 16>(a, s);
      if (nvec <= 32) return short_fwd<TX, TW, V, 32>(a, s);
    }
    if (a.rows_per_group >= 8) {
      if (nvec <= 256) return cols_fwd<TX, TW, V, 1, 256>(a, s);
      if (nvec <= 512) return cols_fwd<TX, TW, V, 2, 256>(a, s);
      if constexpr (V >= 8) {
        if (nvec <= 1024) return cols_fwd<TX, TW, V, 2, 512>(a, s);
      } else {
        if (nvec <= 1024) return cols_fwd<TX, TW, V, 4, 256>(a, s);
        if constexpr (V >= 4) {
          if (nvec <= 2048) return cols_fwd<TX, TW, V, 4, 512>(a, s);
        } else {
          if (nvec <= 2048) return cols_fwd<TX, TW, V, 8, 256>(a, s);
          if (nvec <= 4096) return cols_fwd<TX, TW, V, 8, 512>(a, s);
          if constexpr (V == 1)
            if (nvec <= 8192) return cols_fwd<TX, TW, V, 16, 512>(a, s);
        }
      }
    }
  }
  const int grid = int(a.rows);
  auto threads = [nvec](int nv) { return round_warp((nvec + nv - 1) / nv); };
  // few rows, or a group a row: about 256 threads a row, up to 1024 where the
  // row is longer than 8 vectors (or 16 elements) a thread
  constexpr int kMost = V >= 8 ? 2 : V >= 4 ? 4 : 8;
  if (nvec <= 256)
    norm_fwd_kernel<TX, TW, V, 1><<<grid, threads(1), 0, s>>>(a);
  else if (nvec <= 512)
    norm_fwd_kernel<TX, TW, V, 2><<<grid, threads(2), 0, s>>>(a);
  else if (kMost >= 4 && nvec <= 1024)
    norm_fwd_kernel<TX, TW, V, kMost >= 4 ? 4 : 2><<<grid, threads(4), 0, s>>>(a);
  else if (nvec <= 1024 * kMost)
    norm_fwd_kernel<TX, TW, V, kMost><<<grid, threads(kMost), 0, s>>>(a);
  else
    norm_fwd_long_kernel<TX, TW><<<grid, 1024, 0, s>>>(a);
  return launch_status();
}

template <typename TX, typename TW, int V, int NV, int kThreads>
int row_bwd(const NormBwdArgs& a, int64_t grid, cudaStream_t s) {
  const int thr = round_warp((a.C / V + NV - 1) / NV);
  constexpr size_t stage = size_t(bwd_rows(V * NV)) * 2 * NV * V * sizeof(TX);
  constexpr size_t per = V * sizeof(TX) >= 4 ? bwd_stages(stage) * stage : 0;
  static_assert(per * kThreads <= 200 * 1024, "the rounds of a block fit its shared memory");
  static std::mutex mu;
  static int done[kMaxDevices] = {};
  if (smem_opt_in(done, mu, norm_bwd_kernel<TX, TW, V, NV, kThreads>, per * kThreads) <= 0) {
    cudaGetLastError();
    return PKV_ELAUNCH;
  }
  norm_bwd_kernel<TX, TW, V, NV, kThreads><<<int(grid), thr, per * thr, s>>>(a);
  return launch_status();
}

template <typename TX, typename TW, int V>
int launch_bwd(const NormBwdArgs& a, int64_t groups, cudaStream_t s) {
  const int nvec = a.C / V;
  const int64_t grid = groups * a.parts;
  const int64_t rows = groups * a.rows_per_group;
  if (grid >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  if (nvec <= 192) return row_bwd<TX, TW, V, 1, 192>(a, grid, s);
  if (nvec <= 256) return row_bwd<TX, TW, V, 1, 256>(a, grid, s);
  if (nvec <= 512) return row_bwd<TX, TW, V, 2, 256>(a, grid, s);
  if constexpr (V >= 8) {
    if (nvec <= 1024) return row_bwd<TX, TW, V, 2, 512>(a, grid, s);
  } else {
    if (nvec <= 1024) return row_bwd<TX, TW, V, 4, 256>(a, grid, s);
    if constexpr (V >= 4) {
      if (nvec <= 2048) return row_bwd<TX, TW, V, 4, 512>(a, grid, s);
    } else {
      if (nvec <= 4096) return row_bwd<TX, TW, V, 8, 512>(a, grid, s);
      if constexpr (V == 1)
        if (nvec <= 8192) return row_bwd<TX, TW, V, 16, 512>(a, grid, s);
    }
  }
  // (the column sums first: dx may be in dy's memory)
  const dim3 cols(unsigned(grid), unsigned((a.C + kNormThreads - 1) / kNormThreads));
  if (a.part) norm_cols_kernel<TX><<<cols, kNormThreads, 0, s>>>(a);
  if (a.dx) norm_bwd_long_kernel<TX, TW><<<int(rows), 1024, 0, s>>>(a);
  return launch_status();
}

// Access width: 16 bytes, 4 bytes (16-bit types with even rows), one element.
template <typename TX, typename TW>
int run_fwd(const NormArgs& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(TX);
  auto fits = [&a](int v) {
    const int sx = sizeof(TX), sw = int(sizeof(TW)) * v < 16 ? int(sizeof(TW)) * v : 16;
    return a.C % v == 0 && vec_ok(a.x, a.x_rs, v, sx) && vec_ok(a.y, a.y_rs, v, sx) &&
           vec_ok(a.w, 0, sw, 1) && vec_ok(a.b, 0, sw, 1);
  };
  if (fits(V)) return launch_fwd<TX, TW, V>(a, s);
  if constexpr (sizeof(TX) == 2)
    if (fits(2)) return launch_fwd<TX, TW, 2>(a, s);
  return launch_fwd<TX, TW, 1>(a, s);
}

template <typename TX, typename TW>
int run_bwd(const NormBwdArgs& a, int64_t groups, void* dw, void* db, cudaStream_t s) {
  constexpr int V = 16 / sizeof(TX);
  auto fits = [&a](int v) {
    const int sx = sizeof(TX), sw = int(sizeof(TW)) * v < 16 ? int(sizeof(TW)) * v : 16;
    return a.C % v == 0 && vec_ok(a.x, a.x_rs, v, sx) && vec_ok(a.dy, a.dy_rs, v, sx) &&
           vec_ok(a.dx, a.dx_rs, v, sx) && vec_ok(a.w, 0, sw, 1);
  };
  const bool whole = one_pass(a.parts, a.C);
  NormBwdArgs b = a;
  if (whole) {
    b.part = nullptr;
    b.dw = dw;
    b.db = db;
  }
  int rc = PKV_OK;
  // (short 16-bit rows leave too few threads with 16-byte vectors.  us with those / with
  // 4 bytes, 200 000 rows: 64 columns 86 / 69, 96 90 / 96, 128 86 / 96, 256 90 / 150)
  if (fits(V) && (sizeof(TX) == 4 || a.C >= 128))
    rc = launch_bwd<TX, TW, V>(b, groups, s);
  else if (sizeof(TX) == 2 && fits(2))
    rc = launch_bwd<TX, TW, sizeof(TX) == 2 ? 2 : 1>(b, groups, s);
  else
    rc = launch_bwd<TX, TW, 1>(b, groups, s);
  if (rc != PKV_OK || b.part == nullptr) return rc;
  if (a.C % 4 == 0 && vec_ok(a.part, 0, 16, 1)) {
    const dim3 grid(unsigned(groups), unsigned((a.C + 127) / 128));
    norm_parts_kernel<TW, 4><<<grid, 256, 0, s>>>(a.part, a.parts, a.C, static_cast<TW*>(dw),
                                                  static_cast<TW*>(db));
  } else {
    const dim3 grid(unsigned(groups), unsigned((a.C + 31) / 32));
    norm_parts_kernel<TW, 1><<<grid, 256, 0, s>>>(a.part, a.parts, a.C, static_cast<TW*>(dw),
                                                  static_cast<TW*>(db));
  }
  return launch_status();
}

bool norm_types(int dtype, int wtype) {
  return dtype >= PKV_BF16 && dtype <= PKV_FP32 && (wtype == dtype || wtype == PKV_FP32);
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_layer_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t groups) {
  if (rows <= 0 || cols <= 0 || groups <= 0 || rows % groups != 0) return 0;
  const int64_t parts = bwd_parts(rows / groups, groups, cols);
  return one_pass(parts, cols) ? 0 : groups * parts * 2 * cols * 4;
}

extern "C" int pkv_layer_norm(const void* x, int64_t x_row_stride, const void* weight,
                              const void* bias, int dtype, int wtype, int64_t rows, int64_t cols,
                              int64_t groups, float eps, int one_plus, void* y,
                              int64_t y_row_stride, float* mean, float* rstd,
                              pkv_stream_t stream) {
  if (rows < 0 || cols <= 0 || groups <= 0 || !norm_types(dtype, wtype)) return PKV_EINVAL;
  if (rows == 0) return PKV_OK;
  if (!x || !y || rows % groups != 0 || !(eps >= 0.0f)) return PKV_EINVAL;
  if (cols > kMaxCols || rows >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  NormArgs a{};
  a.x = x;
  a.w = weight;
  a.b = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.x_rs = x_row_stride;
  a.y_rs = y_row_stride;
  a.rows = rows;
  a.rows_per_group = rows / groups;
  a.C = int(cols);
  a.eps = eps;
  a.plus = one_plus ? 1.0f : 0.0f;
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == PKV_BF16)
    return wtype == PKV_FP32 ? run_fwd<__nv_bfloat16, float>(a, s)
                             : run_fwd<__nv_bfloat16, __nv_bfloat16>(a, s);
  if (dtype == PKV_FP16)
    return wtype == PKV_FP32 ? run_fwd<__half, float>(a, s) : run_fwd<__half, __half>(a, s);
  return run_fwd<float, float>(a, s);
}

extern "C" int pkv_layer_norm_backward(const void* dy, int64_t dy_row_stride, const void* x,
                                       int64_t x_row_stride, const void* weight,
                                       const float* mean, const float* rstd, int dtype, int wtype,
                                       int64_t rows, int64_t cols, int64_t groups, int one_plus,
                                       void* dx, int64_t dx_row_stride, void* dweight,
                                       void* dbias, void* workspace, int64_t workspace_bytes,
                                       pkv_stream_t stream) {
  if (rows <= 0 || cols <= 0 || groups <= 0 || !norm_types(dtype, wtype)) return PKV_EINVAL;
  if (!dy || !x || !mean || !rstd || rows % groups != 0) return PKV_EINVAL;
  if (cols > kMaxCols || rows >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (!sums && !dx) return PKV_OK;
  const int64_t need = sums ? pkv_layer_norm_workspace_bytes(rows, cols, groups) : 0;
  if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 4 != 0 ||
                   workspace_bytes < need))
    return PKV_EINVAL;
  NormBwdArgs a{};
  a.dy = dy;
  a.x = x;
  a.w = weight;
  a.mean = mean;
  a.rstd = rstd;
  a.dx = dx;
  a.part = sums ? static_cast<float*>(workspace) : nullptr;
  a.dy_rs = dy_row_stride;
  a.x_rs = x_row_stride;
  a.dx_rs = dx_row_stride;
  a.rows_per_group = rows / groups;
  a.C = int(cols);
  a.parts = int(bwd_parts(rows / groups, groups, cols));
  a.plus = one_plus ? 1.0f : 0.0f;
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == PKV_BF16)
    return wtype == PKV_FP32
               ? run_bwd<__nv_bfloat16, float>(a, groups, dweight, dbias, s)
               : run_bwd<__nv_bfloat16, __nv_bfloat16>(a, groups, dweight, dbias, s);
  if (dtype == PKV_FP16)
    return wtype == PKV_FP32 ? run_bwd<__half, float>(a, groups, dweight, dbias, s)
                             : run_bwd<__half, __half>(a, groups, dweight, dbias, s);
  return run_bwd<float, float>(a, groups, dweight, dbias, s);
}
