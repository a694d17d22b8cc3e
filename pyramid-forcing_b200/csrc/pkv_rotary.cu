// Rotary positions of queries and keys: 1 to 4 position axes, interleaved or
// half pairing, any leading part of the head, fp32 arithmetic.
//
// Pair p < P of a head belongs to axis a = axis[p] and turns by
//   phi = position[token][a] * inv_freq[p]
//   (u, v) -> scale * (u cos phi - v sin phi, u sin phi + v cos phi)
// with (u, v) = elements (2p, 2p + 1) (interleaved) or (p, p + P) (half);
// elements from 2P on are copied.  `inverse` turns by -phi: the transpose,
// which is the gradient's pass.
//
// Bound by HBM: every element is read and written once.  A block owns a few
// tokens: its threads first work out the tokens' cosines and sines once into
// shared memory (the angle is the same in every head of q and of k), then
// stream the heads of q and k through registers in accesses of up to 16
// bytes.  No frequency tables in memory.  The turn count position * inv_freq /
// 2 pi is formed and reduced in pairs of float64 (a position of 10^6 at fp32
// would be off by a tenth of a radian, one of 2^40 in a single float64 by 10^-4),
// and the reduced angle goes through sincospif with its rounding remainder added
// back to first order, so cos and sin are good to fp32's last bit for every
// int64 position while |position * inv_freq| < 2^64.
#include "pkv_vec.cuh"

namespace pkv {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTable = 2048;  // (token, pair) entries of a block's table
constexpr int kRotAxes = 4;

struct RotSide {
  const void* x;
  void* out;
  int64_t x_tok, x_head, o_tok, o_head;
  int heads;
};

// n / d for n < 2^31 by a multiplication (d >= 1): with s = ceil(log2 d) and
// mul = ceil(2^(31 + s) / d) the product's error stays below 1 / d.
struct Div {
  uint32_t mul, shift;
  explicit Div(uint32_t d = 1) {
    shift = 0;
    while ((uint64_t(1) << shift) < d) ++shift;
    mul = uint32_t(((uint64_t(1) << (31 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return uint32_t((uint64_t(n) * mul) >> (31 + shift));
  }
};

struct RotArgs {
  RotSide s[2];
  Div by_heads, by_turn, by_rest;
  int64_t tokens;
  const int64_t* pos;
  const double* inv_freq;
  const int32_t* axis;  // nullptr: one axis
  int n_axes, D, P, half, tile;
  float scale, sign;
};

// Fraction of a turn, [-1/2, 1/2], of n * f radians.  f / 2 pi and its products
// with the halves of n are kept as hi + lo (the rounding error of a product is
// fma(a, b, -a b)); whole turns leave each part before they are added.  Off by
// about 2^-53 + 2^-105 |n f| turns.
__device__ __forceinline__ double turn_fraction(int64_t n, double f) {
  constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;  // 1 / (2 pi)
  const double w = f * kHi, wl = fma(f, kLo, fma(f, kHi, -w));
  const double up = double(n >> 32) * 4294967296.0, dn = double(uint32_t(n));
  const double p = up * w, q = dn * w;
  const double e = fma(up, wl, fma(up, w, -p)) + fma(dn, wl, fma(dn, w, -q));
  const double r = ((p - rint(p)) + (q - rint(q))) + (e - rint(e));
  return r - rint(r);
}

// Eight blocks an SM (32 registers; a few spilled words) keep enough loads on
// their way: 65521 tokens of 24 heads x 128 fp16, a quarter of them turned,
// take 127 us a pass, 806 MB at 6.3 TB/s, 0.97 of the copy rate; with 36
// registers and 7 blocks 133 us, four units a thread at once (80 registers) 222.
// kPair: a unit is V pairs out of two vectors (half layout, and interleaved
// single elements); else it is one vector of V / 2 interleaved pairs.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kRotThreads, V >= 4 ? 8 : 6) rotary_kernel(RotArgs a) {
  constexpr bool kPair = kHalf || V == 1;
  __shared__ float2 tab[kRotTable];
  const int64_t t0 = blockIdx.x * int64_t(a.tile);
  const int nt = int(a.tokens - t0 < a.tile ? a.tokens - t0 : a.tile);
  const int h0 = a.s[0].heads, heads = h0 + a.s[1].heads;
  auto rows = [&](uint32_t th, const T*& x, T*& o, int& t) {
    t = int(a.by_heads.div(th));
    int h = int(th) - t * heads;
    const bool second = h >= h0;
    if (second) h -= h0;
    const RotSide& sd = a.s[second ? 1 : 0];
    x = static_cast<const T*>(sd.x) + (t0 + t) * sd.x_tok + h * sd.x_head;
    o = static_cast<T*>(sd.out) + (t0 + t) * sd.o_tok + h * sd.o_head;
  };
  const int turn = kPair ? a.P / V : 2 * a.P / V;
  const int n = nt * heads * turn;
  for (int i = threadIdx.x; i < nt * a.P; i += kRotThreads) {
    const int t = i / a.P, p = i - t * a.P;
    int ax = a.axis ? a.axis[p] : 0;
    ax = ax < 0 ? 0 : (ax >= a.n_axes ? a.n_axes - 1 : ax);
    const double x = 2.0 * turn_fraction(a.pos[(t0 + t) * a.n_axes + ax], a.inv_freq[p]);
    const float hi = float(x), lo = float(x - double(hi)) * 3.14159265f;
    float s, c;
    sincospif(hi, &s, &c);
    tab[i] = make_float2(fmaf(-lo, s, c) * a.scale, fmaf(lo, c, s) * a.scale * a.sign);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kRotThreads) {
    const uint32_t th = a.by_turn.div(i);
    const int u = i - int(th) * turn;
    const int e = kHalf ? u * V : V == 1 ? 2 * u : u * V;
    const T* x;
    T* o;
    int t;
    rows(th, x, o, t);
    x += e;
    o += e;
    const float2* cs = tab + t * a.P + (kPair ? u * V : u * V / 2);
    if constexpr (kPair) {
      const int gap = kHalf ? a.P : 1;
      float p[V], q[V];
      const Vec<T, V> v0 = ld_vec<T, V>(x), v1 = ld_vec<T, V>(x + gap);
      widen<T, V>(v0, p);
      widen<T, V>(v1, q);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 w = cs[j];
        const float re = p[j] * w.x - q[j] * w.y;
        q[j] = p[j] * w.y + q[j] * w.x;
        p[j] = re;
      }
      st_vec<T, V>(o, narrow<T, V>(p));
      st_vec<T, V>(o + gap, narrow<T, V>(q));
    } else {
      float f[V];
      widen<T, V>(ld_vec<T, V>(x), f);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const float2 w = cs[j / 2];
        const float re = f[j] * w.x - f[j + 1] * w.y;
        f[j + 1] = f[j] * w.y + f[j + 1] * w.x;
        f[j] = re;
      }
      st_vec<T, V>(o, narrow<T, V>(f));
    }
  }
  // copied units of V elements
  const int rest = (a.D - 2 * a.P) / V;
  const int m = nt * heads * rest;
  for (int i = threadIdx.x; i < m; i += kRotThreads) {
    const uint32_t th = a.by_rest.div(i);
    const int e = 2 * a.P + (i - int(th) * rest) * V;
    const T* x;
    T* o;
    int t;
    rows(th, x, o, t);
    st_vec<T, V>(o + e, ld_vec<T, V>(x + e));
  }
}

template <typename T, int V>
bool rot_fits(const RotArgs& a) {
  if ((a.half || V == 1 ? a.P : 2 * a.P) % V || a.D % V) return false;
  for (const RotSide& s : a.s) {
    if (s.heads == 0) continue;
    if (!vec_ok(s.x, s.x_tok, V, sizeof(T)) || !vec_ok(s.out, s.o_tok, V, sizeof(T)) ||
        s.x_head % V || s.o_head % V)
      return false;
  }
  return true;
}

template <typename T, int V>
void launch_rotary(RotArgs a, int64_t grid, cudaStream_t s) {
  a.by_heads = Div(uint32_t(a.s[0].heads + a.s[1].heads));
  const int turn = (a.half || V == 1 ? a.P : 2 * a.P) / V;
  const int rest = (a.D - 2 * a.P) / V;
  if (turn > 0) a.by_turn = Div(uint32_t(turn));
  if (rest > 0) a.by_rest = Div(uint32_t(rest));
  if (a.half)
    rotary_kernel<T, V, true><<<int(grid), kRotThreads, 0, s>>>(a);
  else
    rotary_kernel<T, V, false><<<int(grid), kRotThreads, 0, s>>>(a);
}

template <typename T>
int run_rotary(const RotArgs& a, int64_t grid, cudaStream_t s) {
  // the widest access that divides the pairs, the head, the strides and the
  // addresses
  constexpr int kWide = 16 / sizeof(T);
  if (rot_fits<T, kWide>(a))
    launch_rotary<T, kWide>(a, grid, s);
  else if (kWide > 4 && rot_fits<T, 4>(a))
    launch_rotary<T, 4>(a, grid, s);
  else if (rot_fits<T, 2>(a))
    launch_rotary<T, 2>(a, grid, s);
  else
    launch_rotary<T, 1>(a, grid, s);
  return launch_status();
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_rotary(const void* q, int64_t q_tok_stride, int64_t q_head_stride, int q_heads,
                          void* q_out, int64_t qo_tok_stride, int64_t qo_head_stride,
                          const void* k, int64_t k_tok_stride, int64_t k_head_stride, int k_heads,
                          void* k_out, int64_t ko_tok_stride, int64_t ko_head_stride, int dtype,
                          int64_t tokens, int head_dim, const int64_t* positions, int axes,
                          const double* inv_freq, const int32_t* axis, int pairs, int half,
                          float scale, int inverse, pkv_stream_t stream) {
  if (dtype < PKV_BF16 || dtype > PKV_FP32 || tokens < 0 || q_heads < 0 || k_heads < 0)
    return PKV_EINVAL;
  if (tokens == 0 || q_heads + k_heads == 0) return PKV_OK;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || head_dim <= 0 || pairs < 0 ||
      2 * int64_t(pairs) > head_dim || axes < 1 || axes > kRotAxes ||
      (pairs > 0 && (!positions || !inv_freq || (axes > 1 && !axis))))
    return PKV_EINVAL;
  if (pairs > kRotTable || head_dim > 65536 || q_heads > 65536 || k_heads > 65536)
    return PKV_EUNSUPPORTED;
  RotArgs a{};
  a.s[0] = {q, q_out, q_tok_stride, q_head_stride, qo_tok_stride, qo_head_stride, q_heads};
  a.s[1] = {k, k_out, k_tok_stride, k_head_stride, ko_tok_stride, ko_head_stride, k_heads};
  a.tokens = tokens;
  a.pos = positions;
  a.inv_freq = inv_freq;
  a.axis = axes > 1 ? axis : nullptr;
  a.n_axes = axes;
  a.D = head_dim;
  a.P = pairs;
  a.half = half;
  a.scale = scale;
  a.sign = inverse ? -1.0f : 1.0f;
  // tokens of a block: its table of angles fits, its elements count in 32
  // bits, and there are blocks for every SM
  int64_t tile = pairs > 0 ? kRotTable / pairs : 64;
  const int64_t row = int64_t(q_heads + k_heads) * head_dim;
  const int64_t fill = (tokens + sm_count() * 8 - 1) / (int64_t(sm_count()) * 8);
  if (tile > 8) tile = 8;
  if (tile > fill) tile = fill;
  if (tile < 1) tile = 1;
  // (a thread steps past the last one by up to kRotThreads)
  if (tile * row > INT32_MAX - kRotThreads) return PKV_EUNSUPPORTED;
  a.tile = int(tile);
  const int64_t grid = (tokens + tile - 1) / tile;
  if (grid >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == PKV_BF16) return run_rotary<__nv_bfloat16>(a, grid, s);
  if (dtype == PKV_FP16) return run_rotary<__half>(a, grid, s);
  return run_rotary<float>(a, grid, s);
}
