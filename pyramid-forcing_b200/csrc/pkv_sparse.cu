// Block-sparse attention over the ragged K/V layout: the keys of every
// (chunk, head) segment are cut into blocks of `block` keys, every group of
// `query_block` consecutive query rows of a chunk keeps the top_k blocks whose
// mean key scores highest against the group's summed query, and attends the
// keys of those blocks only.
//
//   mean_j   = sum of the block's keys / their number        (fp32, rounded once)
//   score_gj = (sum over the group's rows of q) . mean_j     (float64)
//   sel_g    = top_k highest scores, equal ones by index, listed ascending, -1 behind
//   out_r    = softmax(scale * q_r . k) v over the keys of sel_g
//
// Its steps:
//  * block_means_kernel -- one pass over K, bound by the conversions to float64
//    and by HBM.  Segment s's block j
//    has row cu[s] / block + s + j of the table: a closed form, so the table
//    needs no offsets of its own (ceil(n / B) <= floor((a + n) / B) - floor(a / B) + 1).
//  * select_blocks_kernel -- scores on the tensor cores with a bound on their
//    error; only blocks within that bound of the last place are scored again in
//    float64 (queries summed in float64, times the fp32 means), so the lists are
//    those of the definition.
//    select_group_kernel -- the same for few groups, in float64 throughout: a
//    mma has 16 rows however few groups share a segment's means.
//  * attention over the listed blocks, by the rows of a group:
//    up to 16 rows (a decoded token, a small group): warps each take 16 keys,
//    K and V go from memory straight into mma fragments, a thread-block
//    cluster splits the list and joins the parts through distributed shared
//    memory -- bound by latency and by the bytes of the listed blocks;
//    more rows: tcgen05 tiles of 128 rows (see sparse_tc_kernel).
#include <cfloat>
#include <mutex>

#include "pkv_internal.h"
#include "pkv_tc.cuh"

namespace pkv {
namespace {

constexpr int kMaxTopK = 1024;
constexpr int kFewRows = 16;  // rows of a group served by the mma kernel

struct SegView {
  int start, len;
};

// Segment s clipped to the K/V rows that exist: a corrupt cu_seqlens reads
// nothing out of range.
__device__ __forceinline__ SegView segment(const int32_t* cu, int s, int64_t kv_rows) {
  const int64_t a = max(cu[s], 0), b = min(int64_t(cu[s + 1]), kv_rows);
  return {int(min(a, kv_rows)), b > a ? int(b - a) : 0};
}

__device__ __forceinline__ uint32_t word(const uint4& w, int i) {
  return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
}

// Eight bf16 elements into float64 sums.  (Four rows at a time added in fp32 first,
// 12% faster, lose low bits where exponents differ by more than 14 and overflow near
// the end of the range; doubles put together by integer operations instead of
// conversions made the means of 2.8 M keys 8% slower.)
__device__ __forceinline__ void add8(double (&acc)[8], const uint4& v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t u = word(v, e);
    acc[2 * e] += double(bf16_bits_to_f32(u & 0xffffu));
    acc[2 * e + 1] += double(__uint_as_float(u & 0xffff0000u));
  }
}

// ---------------------------------------------------------------------------
// Block means
// ---------------------------------------------------------------------------
// W warps a table row (1, or 4 where there are few rows: each then has its
// quarter of the keys on its way at once); 16 (D = 128) or 8 lanes a key, 8
// elements each.  663 000 keys of 128 take 38 us, 4.6 TB/s; 2.8 M keys 130 us, 5.5
// TB/s: the conversions to float64 are what bounds it (34 and 114 us without most
// of them).
template <int D, int W>
__global__ void __launch_bounds__(256)
    block_means_kernel(const uint16_t* __restrict__ k, int64_t kv_rows,
                       const int32_t* __restrict__ cu, int n_seg, int block,
                       float* __restrict__ means, int64_t rows, int zero_rest) {
  constexpr int kLanes = D / 8, kKeys = 32 / kLanes, kRows = 8 / W;  // rows of a block
  __shared__ double part[W > 1 ? 8 : 1][D];
  grid_release();  // the selection may queue up behind this grid
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % W;
  const int sub = lane / kLanes, d0 = (lane % kLanes) * 8;
  const int64_t used = int64_t(cu[n_seg]) / block + n_seg;
  for (int64_t row0 = blockIdx.x * int64_t(kRows); row0 < rows;
       row0 += int64_t(gridDim.x) * kRows) {
    if (row0 >= used && !zero_rest) break;  // (the whole block)
    const int64_t row = row0 + warp / W;
    // last segment whose first row is <= row
    int lo = 0, hi = n_seg - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (int64_t(cu[mid]) / block + mid <= row)
        lo = mid;
      else
        hi = mid - 1;
    }
    const SegView sg = segment(cu, lo, kv_rows);
    const int64_t j = row - (int64_t(cu[lo]) / block + lo);
    const int64_t first = j * block;
    const bool there = row < rows && j >= 0 && first < sg.len;  // a block has this row
    const int n = there ? int(min(int64_t(block), sg.len - first)) : 0;
    const uint16_t* p = k + (sg.start + first) * D + d0;
    double acc[8] = {};
    const int per = block / W, end = min(n, (w + 1) * per);
    for (int r = w * per + sub; r < end; r += 8 * kKeys) {
      uint4 v[8];  // 8 loads a lane on their way: 4 KB a warp
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = r + i * kKeys < end
                   ? __ldg(reinterpret_cast<const uint4*>(p + int64_t(r + i * kKeys) * D))
                   : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) add8(acc, v[i]);
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
    if constexpr (W > 1) {
      if (sub == 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) part[warp][d0 + e] = acc[e];
      __syncthreads();
      if (w == 0 && sub == 0)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          for (int x = 1; x < W; ++x) acc[e] += part[warp + x][d0 + e];
      __syncthreads();
    }
    if (w != 0 || sub != 0 || row >= rows) continue;
    float m[8];
    const bool pow2 = (n & (n - 1)) == 0;  // then the product is exact
    const double inv = 1.0 / double(max(n, 1));
#pragma unroll
    for (int e = 0; e < 8; ++e)
      m[e] = n == 0 ? 0.0f : float(pow2 ? acc[e] * inv : acc[e] / double(n));
    if (there || zero_rest) {
      float* out = means + row * D + d0;
      *reinterpret_cast<float4*>(out) = make_float4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<float4*>(out + 4) = make_float4(m[4], m[5], m[6], m[7]);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(const float* p, uint32_t rank) {
  uint32_t addr;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(su32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Into CTA `rank` of the cluster.
__device__ __forceinline__ void st_cluster(float* p, uint32_t rank, float v) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(su32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Into the cluster's first CTA.
__device__ __forceinline__ void st_leader(uint64_t* p, uint64_t v) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(addr) : "r"(su32(p)));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelGroups = 16;  // groups of a cluster: the rows of an mma
constexpr int kSelCluster = 8;  // most CTAs of one
constexpr int kSelHeld = 16;    // scores a lane of a picking warp keeps in registers
constexpr int kSelChunk = 1024;
static_assert(kMaxTopK + kSelChunk <= 64 * 32, "a lane holds the flags of two tiles of 32");

struct SelectArgs {
  const uint16_t* q;
  int64_t q_rs, q_hs, kv_rows, means_rows;
  const float* means;
  const int32_t* cu;
  int32_t* blocks;
  int H, rows_per_chunk, groups, packs, query_block, block, top_k;
};

// Dynamic shared memory with X CTAs a cluster (kSelGroups / X groups a CTA).
size_t select_bytes(int D, int X, int top_k) {
  const size_t cap = size_t(top_k) + kSelChunk, g = kSelGroups / X;
  return sizeof(double) * (g + kSelWarps) * D + sizeof(float) * kSelGroups * (D + 2) +
         g * cap * 12 + g * top_k * 4;
}

// Scores as integers in the same order; NaN below all, -0 as 0.
__device__ __forceinline__ uint64_t order_key(double s) {
  if (s != s) return 0;
  if (s == 0.0) s = 0.0;
  const int64_t b = __double_as_longlong(s);
  return b < 0 ? ~uint64_t(b) : uint64_t(b) | (uint64_t(1) << 63);
}

// Scores of a picking warp: the first kSelHeld tiles of 32 in registers when
// that is all of them, else in shared memory.
struct Scores {
  float v[kSelHeld];
  const float* s;
  int n;
  bool held;

  __device__ __forceinline__ Scores(const float* scores, int total) : s(scores), n(total) {
    const int lane = threadIdx.x & 31;
    held = n <= 32 * kSelHeld;
#pragma unroll
    for (int t = 0; t < kSelHeld; ++t)
      v[t] = t * 32 + lane < n ? s[t * 32 + lane] : -INFINITY;
  }
  // Scores at or above x.
  __device__ __forceinline__ int at_least(float x) const {
    int c = 0;
    if (held) {
#pragma unroll
      for (int t = 0; t < kSelHeld; ++t) c += __popc(__ballot_sync(0xffffffffu, v[t] >= x));
      return c;
    }
    for (int i = threadIdx.x & 31; i < n; i += 32) c += s[i] >= x;
    return __reduce_add_sync(0xffffffffu, c);
  }
  // Least score at or above x.
  __device__ __forceinline__ float least_from(float x) const {
    float m = INFINITY;
    if (held) {
#pragma unroll
      for (int t = 0; t < kSelHeld; ++t) m = fminf(m, v[t] >= x ? v[t] : INFINITY);
    } else {
      for (int i = threadIdx.x & 31; i < n; i += 32) m = fminf(m, s[i] >= x ? s[i] : INFINITY);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fminf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
  __device__ __forceinline__ float greatest() const {
    float m = -INFINITY;
    if (held) {
#pragma unroll
      for (int t = 0; t < kSelHeld; ++t) m = fmaxf(m, v[t]);
    } else {
      for (int i = threadIdx.x & 31; i < n; i += 32) m = fmaxf(m, s[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
};

// The k-th largest of n > k finite scores, by halving the range until exactly
// k are above (then it is the least of those) or the range is below `close`
// (then its lower end, less than `close` below the k-th).
__device__ __forceinline__ float kth_score(const Scores& sc, int k, float close) {
  float lo = sc.least_from(-FLT_MAX), hi = sc.greatest();
  if (sc.at_least(hi) >= k) return hi;
  while (true) {
    const float mid = 0.5f * lo + 0.5f * hi;
    if (!(mid > lo && mid < hi) || hi - lo < close) return lo;
    const int c = sc.at_least(mid);
    if (c == k) return sc.least_from(mid);
    if (c > k)
      lo = mid;
    else
      hi = mid;
  }
}

// Two fp32 values as bf16 pairs, hi + lo: 16 bits of each.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x, y);
  lo = pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// A cluster of X CTAs serves 16 groups of a segment: each CTA sums the queries
// of its share of the groups (group i belongs to rank i % X), all of them score
// their share of the blocks for all 16 groups on mma.m16n8k16 (rows = groups,
// columns = blocks), hand the scores to the groups' owners through distributed
// shared memory, and every CTA picks for its groups.  A block's mean is read
// once for 16 groups, and a single token's table by many SMs.
//
// Operands are split into bf16 hi + lo and multiplied as hi hi + hi lo + lo hi.
// For x in [1, 2) hi is off by at most 2^-8 and lo, at most 2^-8, by 2^-17: the
// product of two such loses at most 2^-16 (lo lo) + 2 * 2^-17, 8 * 2^-18 of |x y|,
// and by Cauchy and Schwarz a score 8 * 2^-18 |q| |mean|.  Accumulation: 4 mma of 17
// addends in a chain; with each addend cut off below 2^-22 of the largest (an
// assumption with two bits to spare over 24-bit sums) at most 68 * 2^-22 = 4.3 *
// 2^-18 of it; the summed query in fp32 and the sums of the chains stay below
// 0.1 * 2^-18.  So e = 2^-14 |q| |mean| = 16 * 2^-18 bounds the error 1.29 times over
// (1.75 times if addends are cut off at 2^-24).  With T the top_k-th such score, a
// block above T + 2 e is in the list for certain and one below T - 2 e is not; those
// between are scored in float64 and ranked, unless all of them are in.  Infinite or
// NaN queries or means make every block such a one, and so do |q| |mean| whose
// products could pass fp32's range: with scores of infinity T + 2 e would be
// infinite, and more than top_k blocks could be above it.
//   468 groups over 36 segments of 73 to 512 blocks take 20 us, 1872 groups over
// 144 segments 47; float64 scores by a CTA a group took 26 and 73.  Latency: loads,
// cluster barriers, one warp's pick; issue slots 20% busy.  Where all scores of the
// groups are near (zero queries, an infinite mean in every segment) the first takes
// 80 to 100 us.
template <int D, int X>
__global__ void __launch_bounds__(kSelThreads, 2) select_blocks_kernel(SelectArgs a) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kMine = kSelGroups / X;  // groups a CTA owns
  constexpr int kQs = D + 2;             // row stride of qf: no bank conflicts
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ float nmax[kSelCluster * kSelWarps];
  const int cap = a.top_k + kSelChunk;
  double* qs = reinterpret_cast<double*>(raw);                     // [kMine][D] summed queries
  double* red = qs + kMine * D;                                    // [warps][D]
  uint64_t* exact = reinterpret_cast<uint64_t*>(red + kSelWarps * D);  // [kMine][cap] float64
  float* qf = reinterpret_cast<float*>(exact + kMine * cap);       // [16][D + 2] of all groups
  float* score = qf + kSelGroups * kQs;                            // [kMine][cap]
  int* kid = reinterpret_cast<int*>(score + kMine * cap);          // [kMine][top_k] kept earlier
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_wait();  // (from here on plain loads: the read-only path is for data that no
                // kernel still running when this one started has written)
  grid_release();  // the attention may queue up behind this grid
  const int rank = int(cluster_rank());
  const int unit = blockIdx.x / X;
  const int s = unit / a.packs, g0 = (unit - s * a.packs) * kSelGroups;
  const int ng = min(kSelGroups, a.groups - g0);
  const int c = s / a.H, h = s - c * a.H;
  const SegView sg = segment(a.cu, s, a.kv_rows);
  const int nblk = (sg.len + a.block - 1) / a.block;
  int32_t* out = a.blocks + (int64_t(s) * a.groups + g0) * a.top_k;  // ng lists
  if (nblk <= a.top_k) {  // every block is kept (the whole cluster leaves)
    for (int i = rank * kSelThreads + tid; i < ng * a.top_k; i += X * kSelThreads) {
      const int j = i % a.top_k;
      out[i] = j < nblk ? j : -1;
    }
    return;
  }
  // ---- sums of this CTA's groups' queries in float64 ----
  for (int i = tid; i < (kSelGroups - ng) * kQs; i += kSelThreads) qf[ng * kQs + i] = 0.0f;
  {
    constexpr int kLanes = D / 8, kPerWarp = 32 / kLanes, kWarps = kSelWarps / kMine;
    constexpr int kRows = kWarps * kPerWarp;
    const int g = warp / kWarps * X + rank;
    const int sub = warp % kWarps * kPerWarp + lane / kLanes, d0 = (lane % kLanes) * 8;
    const int r0 = (g0 + g) * a.query_block;
    const int nr = g < ng ? min(a.query_block, a.rows_per_chunk - r0) : 0;
    const uint16_t* p =
        a.q + (int64_t(c) * a.rows_per_chunk + r0) * a.q_rs + int64_t(h) * a.q_hs + d0;
    double acc[8] = {};
    for (int r = sub; r < nr; r += 16 * kRows) {
      uint4 v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = r + i * kRows < nr
                   ? *reinterpret_cast<const uint4*>(p + int64_t(r + i * kRows) * a.q_rs)
                   : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) add8(acc, v[i]);
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(kAll, acc[e], o);
    if (lane < kLanes)
#pragma unroll
      for (int e = 0; e < 8; ++e) red[warp * D + d0 + e] = acc[e];
    cluster_barrier();  // the other CTAs run: their memory may be written
    for (int i = tid; i < kMine * D; i += kSelThreads) {
      double t = 0.0;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) t += red[(i / D * kWarps + x) * D + i % D];
      qs[i] = t;
      const int gi = i / D * X + rank;
      if (gi < ng)
#pragma unroll
        for (int x = 0; x < X; ++x) st_cluster(&qf[gi * kQs + i % D], x, float(t));
    }
  }
  cluster_barrier();
  // ---- queries as A fragments: with lane (g, c) = (lane / 4, lane % 4),
  // k-steps 2i, 2i + 1 take dims 32 i + 8 c .. + 7 (the order of the
  // contraction is free), so a mean's lanes load 32 bytes each ----
  const int gr = lane >> 2, cc = lane & 3;
  uint32_t ah[D / 32][8], al[D / 32][8];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
      const float* p = qf + (gr + 8 * hrow) * kQs + 32 * i + 8 * cc;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 w = *reinterpret_cast<const float2*>(p + 2 * e);
        split2(w.x, w.y, ah[i][2 * e + hrow], al[i][2 * e + hrow]);
      }
    }
  const int64_t base = int64_t(a.cu[s]) / a.block + s;
  int kept = 0;
  float most = 0.0f;  // largest |mean|^2 that this warp has seen
  for (int b0 = 0; b0 < nblk; b0 += kSelChunk) {
    const int m = min(kSelChunk, nblk - b0);
    for (int t = rank * kSelWarps + warp; t * 8 < m; t += X * kSelWarps) {
      const int64_t row = base + b0 + t * 8 + gr;
      const bool ok = t * 8 + gr < m && row >= 0 && row < a.means_rows;
      const float* p = a.means + row * D + 8 * cc;
      float4 f[D / 32][2];
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          f[i][e] = ok ? *reinterpret_cast<const float4*>(p + 32 * i + 4 * e)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
      float part[4][4] = {};  // independent chains of mma
      float n2 = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 v = f[i][e];
          n2 = fmaf(v.x, v.x, fmaf(v.y, v.y, fmaf(v.z, v.z, fmaf(v.w, v.w, n2))));
          uint32_t bh0, bl0, bh1, bl1;
          split2(v.x, v.y, bh0, bl0);
          split2(v.z, v.w, bh1, bl1);
          const uint32_t* x = ah[i] + 4 * e;
          const uint32_t* y = al[i] + 4 * e;
          mma_16816(part[0], y[0], y[1], y[2], y[3], bh0, bh1);
          mma_16816(part[1], x[0], x[1], x[2], x[3], bl0, bl1);
          mma_16816(part[2 + e], x[0], x[1], x[2], x[3], bh0, bh1);
        }
      n2 += __shfl_xor_sync(kAll, n2, 1);
      n2 += __shfl_xor_sync(kAll, n2, 2);
      most = n2 < INFINITY ? fmaxf(most, n2) : INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int gi = gr + 8 * (e >> 1), i = t * 8 + 2 * cc + (e & 1);
        const float v = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
        if (gi < ng && i < m) st_cluster(&score[gi / X * cap + kept + i], gi % X, v);
      }
    }
    float all_most = most;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) all_most = fmaxf(all_most, __shfl_xor_sync(kAll, all_most, o));
    if (lane < X) st_cluster(&nmax[rank * kSelWarps + warp], lane, all_most);
    cluster_barrier();  // the scores of this CTA's groups are here
    const int total = kept + m;
    const bool last = b0 + m == nblk;
    // ---- pick: a warp a group ----
    for (int g = warp; g < kMine && g * X + rank < ng; g += kSelWarps) {
      int* kd = kid + g * a.top_k;
      if (total <= a.top_k) {  // (not the last round)
        for (int i = lane; i < m; i += 32) kd[kept + i] = b0 + i;
        continue;
      }
      int32_t* list = out + int64_t(g * X + rank) * a.top_k;
      float* sc = score + g * cap;
      uint64_t* ex = exact + g * cap;
      const double* qg = qs + g * D;
      double qn = 0.0;
#pragma unroll
      for (int d = 0; d < D; d += 32) qn = fma(qg[d + lane], qg[d + lane], qn);
      float mm = 0.0f;
      for (int i = lane; i < X * kSelWarps; i += 32) mm = fmaxf(mm, nmax[i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        qn += __shfl_xor_sync(kAll, qn, o);
        mm = fmaxf(mm, __shfl_xor_sync(kAll, mm, o));
      }
      // 2.25 e, rounded up: T may be 0.1 e2 low, so 2 e + 0.1 e2 <= e2 has to hold,
      // e2 >= 2.23 e; the addend covers parts that underflow
      const float ql = sqrtf(float(qn)), ml = sqrtf(mm);
      const float e2 = 2.25f * 6.103515625e-5f * 1.001f * ql * ml + 1e-35f * (ql + ml) + 1e-36f;
      // (|q| |mean| bounds the products and their partial sums, which must be finite)
      const bool all =
          !(e2 < INFINITY) || !(ql * ml < 1e37f) || !(ql > 1e-15f) || !(ml > 1e-15f);
      const Scores held(sc, total);
      float lo = -INFINITY, hi = INFINITY;
      int nsure = 0, nnear = total;
      if (!all) {
        // (T may be 0.1 e2 below the top_k-th: the margin of 2.25 covers it)
        const float T = kth_score(held, a.top_k, 0.1f * e2);
        lo = T - e2;
        hi = T + e2;
        nsure = held.at_least(hi);
        nnear = held.at_least(lo) - nsure;
      }
      // near: at least lo (or all) and below hi
      auto is_near = [&](float x) { return all || (x >= lo && x < hi); };
      const int need = a.top_k - nsure;
      // exact score of the block at index j of the present scores
      auto score64 = [&](int j) {
        const int64_t row = base + (j < kept ? kd[j] : b0 + j - kept);
        double x = 0.0;
        if (row >= 0 && row < a.means_rows)
#pragma unroll
          for (int d = 0; d < D; d += 32)
            x = fma(double(a.means[row * D + d + lane]), qg[d + lane], x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
        return order_key(x);
      };
      if (!all && held.held && kept == 0 && last && nnear <= 32) {
        // ---- the usual case: scores in registers, few near ones.  Bit p of
        // `in`: the p-th near one is in the list ----
        uint32_t in = 0xffffffffu;
        if (nnear > need) {
          int* idx = reinterpret_cast<int*>(ex);  // the near ones' indices
          int at = 0;
#pragma unroll
          for (int t = 0; t < kSelHeld; ++t) {
            const bool is = is_near(held.v[t]);
            const uint32_t nb = __ballot_sync(kAll, is);
            if (is) idx[at + __popc(nb & ((1u << lane) - 1))] = t * 32 + lane;
            at += __popc(nb);
          }
          __syncwarp();
          uint64_t mine = 0;  // lane p: the p-th one's score
          for (int p = 0; p < nnear; ++p) {
            const uint64_t x = score64(idx[p]);
            if (lane == p) mine = x;
          }
          int ahead = 0;
          for (int p = 0; p < nnear; ++p) {
            const uint64_t x = __shfl_sync(kAll, mine, p);
            ahead += x > mine || (x == mine && p < lane);
          }
          in = __ballot_sync(kAll, lane < nnear && ahead < need);
        }
        int at = 0, seen = 0;
#pragma unroll
        for (int t = 0; t < kSelHeld; ++t) {
          const uint32_t below = (1u << lane) - 1;
          const bool is = is_near(held.v[t]);
          const uint32_t nb = __ballot_sync(kAll, is);
          const bool keep = held.v[t] >= hi || (is && (in >> (seen + __popc(nb & below)) & 1));
          const uint32_t kb = __ballot_sync(kAll, keep);
          if (keep) list[at + __popc(kb & below)] = t * 32 + lane;
          at += __popc(kb);
          seen += __popc(nb);
        }
        continue;
      }
      // ---- float64 scores of the near ones, in index order: a lane a block where
      // there are many, the warp a block else (either adds in its own order, so one
      // of them for all).  Of those, `bar` and the first `ties` at it are kept ----
      uint64_t bar = 0;
      int ties = need;
      if (nnear > need) {
        uint64_t mn = ~uint64_t(0), mx = 0;
        int at = 0;
        for (int t0 = 0; t0 < total; t0 += 32) {
          const int i = t0 + lane;
          const bool is = i < total && is_near(sc[i]);
          uint32_t todo = __ballot_sync(kAll, is);
          const int to = at + __popc(todo & ((1u << lane) - 1));
          at += __popc(todo);
          uint64_t mine = 0;
          if (nnear > 32) {
            const int64_t row = base + (i < kept ? kd[i] : b0 + i - kept);
            double x[4] = {};
            if (is && row >= 0 && row < a.means_rows)
#pragma unroll 4
              for (int d = 0; d < D; d += 4) {
                const float4 m = *reinterpret_cast<const float4*>(a.means + row * D + d);
                x[0] = fma(double(m.x), qg[d], x[0]);
                x[1] = fma(double(m.y), qg[d + 1], x[1]);
                x[2] = fma(double(m.z), qg[d + 2], x[2]);
                x[3] = fma(double(m.w), qg[d + 3], x[3]);
              }
            mine = order_key((x[0] + x[1]) + (x[2] + x[3]));
          } else {
            while (todo) {
              const int l = __ffs(todo) - 1;
              todo &= todo - 1;
              const uint64_t x = score64(t0 + l);
              if (lane == l) mine = x;
            }
          }
          if (is) {
            ex[to] = mine;
            mn = min(mn, mine);
            mx = max(mx, mine);
          }
        }
        __syncwarp();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          mn = min(mn, __shfl_xor_sync(kAll, mn, o));
          mx = max(mx, __shfl_xor_sync(kAll, mx, o));
        }
        // the need-th highest bit by bit, from the highest that differs
        auto count = [&](uint64_t x) {
          int c = 0;
          for (int i = lane; i < nnear; i += 32) c += ex[i] >= x;
          return __reduce_add_sync(kAll, c);
        };
        int bit = mn == mx ? -1 : 63 - __clzll(mn ^ mx);
        bar = bit < 0 ? mx : bit == 63 ? 0 : mx >> (bit + 1) << (bit + 1);
        for (; bit >= 0; --bit) {
          const uint64_t x = bar | uint64_t(1) << bit;
          const int c = count(x);
          if (c >= need) bar = x;
          if (c == need) break;
        }
        ties = need - (bar == ~uint64_t(0) ? 0 : count(bar + 1));
      }
      // ---- which to keep.  Lane t holds the flags of tiles t and t + 32 ----
      uint32_t flags[2] = {0, 0};
      int seen = 0, even = 0;  // near ones so far, and those at the bar
      for (int t0 = 0; t0 < total; t0 += 32) {
        const uint32_t below = (1u << lane) - 1;
        const int i = t0 + lane;
        const float v = i < total ? sc[i] : -INFINITY;
        const bool is = i < total && is_near(v);
        bool keep = !all && i < total && v >= (nnear > need ? hi : lo);
        if (nnear > need) {
          const uint32_t nb = __ballot_sync(kAll, is);
          const uint64_t x = is ? ex[seen + __popc(nb & below)] : 0;
          const uint32_t eb = __ballot_sync(kAll, is && x == bar);
          keep = keep || (is && (x > bar || (x == bar && even + __popc(eb & below) < ties)));
          seen += __popc(nb);
          even += __popc(eb);
        }
        const uint32_t kb = __ballot_sync(kAll, keep);
        if (lane == ((t0 >> 5) & 31)) (t0 < 1024 ? flags[0] : flags[1]) = kb;
      }
      // ---- move them up, in index order ----
      int at = 0;
      for (int t0 = 0; t0 < total; t0 += 32) {
        const int i = t0 + lane;
        const uint32_t kb = __shfl_sync(kAll, t0 < 1024 ? flags[0] : flags[1], (t0 >> 5) & 31);
        const bool keep = kb >> lane & 1;
        const int to = at + __popc(kb & ((1u << lane) - 1));
        const int id = keep ? (i < kept ? kd[i] : b0 + i - kept) : 0;
        if (last) {
          if (keep) list[to] = id;
        } else {
          const float v = keep ? sc[i] : 0.0f;
          __syncwarp();
          if (keep) {
            sc[to] = v;
            kd[to] = id;
          }
          __syncwarp();
        }
        at += __popc(kb);
      }
    }
    kept = min(total, a.top_k);
    if (last) return;
    cluster_barrier();  // every CTA has picked: its memory may be written
  }
}

struct GroupSmem {
  double red[kSelThreads / 32][128];  // the warps' query sums
  double q[128];
  int hist[256];
  int wsum[2][kSelThreads / 32];
  uint64_t prefix, lo, hi;
  int need, done;
  // [top_k + kSelChunk] keys, then as many ids: the kept blocks of earlier
  // rounds, then the present one's
  uint64_t key[1];
};

// The form for few groups: a CTA a group, or a cluster whose CTAs share the
// scores and whose first picks.  Scores are float64 products straight away, and
// the pick goes by the scores' digits, 8 bits at a time.
template <int D>
__global__ void __launch_bounds__(kSelThreads, 4) select_group_kernel(SelectArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  GroupSmem& sm = *reinterpret_cast<GroupSmem*>(raw);
  uint64_t* skey = sm.key;
  int* sid = reinterpret_cast<int*>(skey + a.top_k + kSelChunk);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int X = int(cluster_size()), rank = int(cluster_rank());
  grid_wait();  // (and plain loads from here on, as in the kernel above)
  grid_release();
  const int unit = blockIdx.x / X;
  const int s = unit / a.groups, g = unit - s * a.groups;
  const int c = s / a.H, h = s - c * a.H;
  const SegView sg = segment(a.cu, s, a.kv_rows);
  const int nblk = (sg.len + a.block - 1) / a.block;
  int32_t* out = a.blocks + int64_t(unit) * a.top_k;
  if (nblk <= a.top_k) {  // every block is kept (the whole cluster leaves)
    if (rank == 0)
      for (int i = tid; i < a.top_k; i += kSelThreads) out[i] = i < nblk ? i : -1;
    return;
  }
  // ---- sum of the group's queries in float64 ----
  const int r0 = g * a.query_block;
  const int nr = min(a.query_block, a.rows_per_chunk - r0);
  {
    constexpr int kLanes = D / 8, kRows = kSelThreads / kLanes;
    const int sub = tid / kLanes, d0 = (tid % kLanes) * 8;
    const uint16_t* p =
        a.q + (int64_t(c) * a.rows_per_chunk + r0) * a.q_rs + int64_t(h) * a.q_hs + d0;
    double acc[8] = {};
    for (int r = sub; r < nr; r += 4 * kRows) {
      uint4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = r + i * kRows < nr
                   ? *reinterpret_cast<const uint4*>(p + int64_t(r + i * kRows) * a.q_rs)
                   : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) add8(acc, w[i]);
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
    if (lane < kLanes)
#pragma unroll
      for (int e = 0; e < 8; ++e) sm.red[warp][d0 + e] = acc[e];
    __syncthreads();
    if (tid < D) {
      double t = 0.0;
#pragma unroll
      for (int i = 0; i < kSelThreads / 32; ++i) t += sm.red[i][tid];
      sm.q[tid] = t;
    }
    __syncthreads();
  }
  // ---- scores: 16 lanes a block, D / 16 products each; 4 blocks on their way ----
  constexpr int kPer = D / 16, kVec = kPer / 4, kBatch = 4;
  const int l16 = tid & 15;
  double q[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) q[i] = sm.q[(i / 4) * 64 + l16 * 4 + (i & 3)];
  const int64_t base = int64_t(a.cu[s]) / a.block + s;
  const int stride = X * (kSelThreads / 16);
  int kept = 0;
  if (X > 1) cluster_barrier();  // the first CTA runs: its memory may be written
  for (int b0 = 0; b0 < nblk; b0 += kSelChunk) {
    const int m = min(kSelChunk, nblk - b0);
    uint64_t mn = ~uint64_t(0), mx = 0;
    for (int i0 = rank * (kSelThreads / 16) + (tid >> 4); i0 < kSelChunk; i0 += stride * kBatch) {
      if (i0 - (lane >> 4) >= m) break;  // (the whole warp)
      float4 f[kBatch][kVec];
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const int64_t row = base + b0 + i0 + x * stride;
        const bool ok = i0 + x * stride < m && row >= 0 && row < a.means_rows;
        const float* p = a.means + row * D + l16 * 4;
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          f[x][e] = ok ? *reinterpret_cast<const float4*>(p + e * 64)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        double t = 0.0;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          t = fma(double(f[x][e].x), q[4 * e], t);
          t = fma(double(f[x][e].y), q[4 * e + 1], t);
          t = fma(double(f[x][e].z), q[4 * e + 2], t);
          t = fma(double(f[x][e].w), q[4 * e + 3], t);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        const int i = i0 + x * stride;
        if (i < m && l16 == 0) st_leader(&skey[kept + i], order_key(t));
      }
    }
    if (rank == 0)
      for (int i = tid; i < m; i += kSelThreads) sid[kept + i] = b0 + i;
    if (X > 1)
      cluster_barrier();  // every score is in the first CTA's memory
    else
      __syncthreads();
    const int total = kept + m;
    const bool last = b0 + m == nblk;
    if (rank != 0) {
      if (last) return;
      kept = min(total, a.top_k);
      cluster_barrier();  // the first CTA has picked: its memory may be written
      continue;
    }
    if (total <= a.top_k) {  // (not the last round: nblk > top_k)
      kept = total;
      if (X > 1) cluster_barrier();
      continue;
    }
    // ---- the top_k-th key: digits of 8 bits from the highest that differs ----
    for (int i = tid; i < total; i += kSelThreads) {
      mn = min(mn, skey[i]);
      mx = max(mx, skey[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (tid == 0) {
      sm.lo = ~uint64_t(0);
      sm.hi = 0;
    }
    __syncthreads();
    if (lane == 0) {
      atomicMin(reinterpret_cast<unsigned long long*>(&sm.lo), mn);
      atomicMax(reinterpret_cast<unsigned long long*>(&sm.hi), mx);
    }
    __syncthreads();
    mn = sm.lo;
    mx = sm.hi;
    int shift = mn == mx ? 0 : 64 - __clzll(mn ^ mx);  // bits below `shift` differ
    uint64_t prefix = shift == 64 ? 0 : mx >> shift;
    int need = a.top_k;
    bool exact = false;  // every key with the prefix is kept
    while (shift > 0 && !exact) {
      const int bits = min(8, shift);
      shift -= bits;
      for (int i = tid; i < 256; i += kSelThreads) sm.hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < total; i += kSelThreads) {
        const uint64_t key = skey[i];
        const uint64_t up = shift + bits == 64 ? 0 : key >> (shift + bits);
        if (up == prefix) atomicAdd(&sm.hist[int(key >> shift) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      if (warp == 0) {
        // lane owns bins 255 - 8 lane .. 248 - 8 lane: a scan from the top
        int cnt[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += cnt[i] = sm.hist[255 - 8 * lane - i];
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += y;
        }
        before -= sum;
        if (before < need && before + sum >= need) {
          int acc = before;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (acc < need && acc + cnt[i] >= need) {
              sm.prefix = (prefix << bits) | uint64_t(255 - 8 * lane - i);
              sm.need = need - acc;
              sm.done = cnt[i] == need - acc;
            }
            acc += cnt[i];
          }
        }
      }
      __syncthreads();
      prefix = sm.prefix;
      need = sm.need;
      exact = sm.done != 0;
      __syncthreads();
    }
    // ---- keep: above the prefix, and the first `need` at it, in index order ----
    int eq_seen = 0, written = 0;
    for (int t0 = 0; t0 < total; t0 += kSelThreads) {
      const int i = t0 + tid;
      const uint64_t key = i < total ? skey[i] : 0;
      const int id = i < total ? sid[i] : 0;
      const uint64_t up = shift == 64 ? 0 : key >> shift;
      const bool gt = i < total && up > prefix, eq = i < total && up == prefix;
      const uint32_t be = __ballot_sync(0xffffffffu, eq);
      if (lane == 0) sm.wsum[0][warp] = __popc(be);
      __syncthreads();
      int er = eq_seen + __popc(be & ((1u << lane) - 1));
      for (int w = 0; w < kSelThreads / 32; ++w) {
        if (w < warp) er += sm.wsum[0][w];
        eq_seen += sm.wsum[0][w];
      }
      const bool keep = gt || (eq && er < need);
      const uint32_t bk = __ballot_sync(0xffffffffu, keep);
      if (lane == 0) sm.wsum[1][warp] = __popc(bk);
      __syncthreads();
      int at = written + __popc(bk & ((1u << lane) - 1));
      for (int w = 0; w < kSelThreads / 32; ++w) {
        if (w < warp) at += sm.wsum[1][w];
        written += sm.wsum[1][w];
      }
      // at <= i, and every key of this tile is in registers: in place
      if (keep && at < a.top_k) {
        if (last)
          out[at] = id;
        else {
          skey[at] = key;
          sid[at] = id;
        }
      }
      __syncthreads();
    }
    kept = a.top_k;
    if (X > 1 && !last) cluster_barrier();
  }
}

// ---------------------------------------------------------------------------
// Attention of up to 16 rows
// ---------------------------------------------------------------------------
struct SparseArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_rs, q_hs, kv_rows, o_rs, o_hs;
  const int32_t* cu;
  const int32_t* blocks;
  uint16_t* out;
  int32_t* status;
  int H, rows_per_chunk, groups, query_block, block, top_k;
  float scale_log2;
};

constexpr int kFewWarps = 8;

// Partial results of the warps and of the CTA: unnormalised O, maximum, sum.
template <int D>
struct FewSmem {
  float o[kFewWarps][kFewRows][D];
  float m[kFewWarps][kFewRows], l[kFewWarps][kFewRows];
  float co[kFewRows][D];
  float cm[kFewRows], cl[kFewRows];
  int list[kMaxTopK];
  int count;
};

// A cluster a (segment, group); its warps take chunks of 16 keys of the listed
// blocks in turn.  With the fragment layout of mma.m16n8k16 a lane (g, c) =
// (lane / 4, lane % 4) holds, of a tile of 8 keys, key g and two dim pairs per
// k-step.  The order of the contraction is free, so k-steps 2i, 2i + 1 take
// dims 32 i + 8 c .. + 7: one 16-byte load a key and 32 dims, for Q alike.  For
// P V, lane (g, c) holds keys 2c, 2c + 1, 2c + 8, 2c + 9 of column g of an
// output tile; columns are free too, so tile t takes dim 8 g + t: four
// 16-byte loads of V rows serve 8 tiles after pairing the halves of two keys.
//   12 rows of 16 blocks of 64 take 7 us, latency from the list to the join.  Every
// group reads its own keys: 1560 rows of 36 heads with a list a row take 7.8 ms
// (59 GB through L2), with a list for 16 rows 0.73 ms.
template <int D>
__global__ void __launch_bounds__(kFewWarps * 32) sparse_few_kernel(SparseArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  FewSmem<D>& sm = *reinterpret_cast<FewSmem<D>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_wait();  // (plain loads from here on, of K and V too: the kernel before this one
                // may be what wrote them, and may have let this one start early)
  const int X = int(cluster_size()), rank = int(cluster_rank());
  const int unit = blockIdx.x / X;
  const int s = unit / a.groups, grp = unit - s * a.groups;
  const int ch = s / a.H, h = s - ch * a.H;
  const int r0 = grp * a.query_block;
  const int nr = min(a.query_block, a.rows_per_chunk - r0);
  const SegView sg = segment(a.cu, s, a.kv_rows);
  const int nblk = (sg.len + a.block - 1) / a.block;
  const int g = lane >> 2, c = lane & 3;
  // ---- the listed blocks that exist, in order ----
  if (warp == 0) {
    const int32_t* lst = a.blocks + int64_t(unit) * a.top_k;
    int n = 0;
    for (int b = 0; b < a.top_k; b += 32) {
      const int e = b + lane < a.top_k ? lst[b + lane] : -1;
      const bool ok = e >= 0 && e < nblk;
      const uint32_t m = __ballot_sync(0xffffffffu, ok);
      if (ok) sm.list[n + __popc(m & ((1u << lane) - 1))] = e;
      n += __popc(m);
    }
    if (lane == 0) sm.count = n;
  }
  // ---- queries as A fragments ----
  const uint16_t* qp =
      a.q + (int64_t(ch) * a.rows_per_chunk + r0) * a.q_rs + int64_t(h) * a.q_hs;
  uint4 q0[D / 32], q1[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    q0[i] = g < nr ? *reinterpret_cast<const uint4*>(qp + g * a.q_rs + 32 * i + 8 * c)
                   : make_uint4(0, 0, 0, 0);
    q1[i] = g + 8 < nr ? *reinterpret_cast<const uint4*>(qp + (g + 8) * a.q_rs + 32 * i + 8 * c)
                       : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  const int per = a.block / 16;
  const int chunks = sm.count * per;
  float o[D / 8][4];
#pragma unroll
  for (int t = 0; t < D / 8; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  for (int i = rank * kFewWarps + warp; i < chunks; i += X * kFewWarps) {
    const int key0 = sm.list[i / per] * a.block + (i % per) * 16;
    const int valid = sg.len - key0;  // keys of this chunk inside the segment
    if (valid <= 0) continue;
    const uint16_t* kp = a.k + (int64_t(sg.start) + key0) * D;
    const uint16_t* vp = a.v + (int64_t(sg.start) + key0) * D;
    uint4 kw[2][D / 32], vw[4][D / 64];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < D / 32; ++e)
        kw[t][e] = t * 8 + g < valid
                       ? *reinterpret_cast<const uint4*>(kp + (t * 8 + g) * D + 32 * e + 8 * c)
                       : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int key = 2 * c + (t & 1) + (t >> 1) * 8;
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        vw[t][e] = key < valid
                       ? *reinterpret_cast<const uint4*>(vp + key * D + 64 * e + 8 * g)
                       : make_uint4(0, 0, 0, 0);
    }
    float sc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) {
        mma_16816(sc[t], q0[e].x, q1[e].x, q0[e].y, q1[e].y, kw[t][e].x, kw[t][e].y);
        mma_16816(sc[t], q0[e].z, q1[e].z, q0[e].w, q1[e].w, kw[t][e].z, kw[t][e].w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sc[t][e] = t * 8 + 2 * c + (e & 1) < valid ? sc[t][e] * a.scale_log2 : -INFINITY;
    }
    float n0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
    float n1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
      n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
    }
    n0 = fmaxf(n0, m0);
    n1 = fmaxf(n1, m1);
    // a row whose scores are all -inf keeps a reference of 0
    const float u0 = n0 == -INFINITY ? 0.0f : n0, u1 = n1 == -INFINITY ? 0.0f : n1;
    const float f0 = fast_exp2(m0 - u0), f1 = fast_exp2(m1 - u1);
    m0 = n0;
    m1 = n1;
    float p[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      p[t][0] = fast_exp2(sc[t][0] - u0);
      p[t][1] = fast_exp2(sc[t][1] - u0);
      p[t][2] = fast_exp2(sc[t][2] - u1);
      p[t][3] = fast_exp2(sc[t][3] - u1);
    }
    l0 = l0 * f0 + ((p[0][0] + p[0][1]) + (p[1][0] + p[1][1]));
    l1 = l1 * f1 + ((p[0][2] + p[0][3]) + (p[1][2] + p[1][3]));
#pragma unroll
    for (int t = 0; t < D / 8; ++t) {
      o[t][0] *= f0;
      o[t][1] *= f0;
      o[t][2] *= f1;
      o[t][3] *= f1;
    }
    // P is rounded to bf16 for the product, as the tile kernel's is: half a
    // step of 2^-8 a weight, averaged over the keys
    const uint32_t a0 = pack_bf16x2(p[0][0], p[0][1]), a1 = pack_bf16x2(p[0][2], p[0][3]);
    const uint32_t a2 = pack_bf16x2(p[1][0], p[1][1]), a3 = pack_bf16x2(p[1][2], p[1][3]);
#pragma unroll
    for (int e = 0; e < D / 64; ++e)
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t sel = (t & 1) ? 0x7632u : 0x5410u;
        const uint32_t b0 = __byte_perm(word(vw[0][e], t >> 1), word(vw[1][e], t >> 1), sel);
        const uint32_t b1 = __byte_perm(word(vw[2][e], t >> 1), word(vw[3][e], t >> 1), sel);
        mma_16816(o[e * 8 + t], a0, a1, a2, a3, b0, b1);
      }
  }
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  // ---- join the warps ----
  if (c == 0) {
    sm.m[warp][g] = m0;
    sm.m[warp][g + 8] = m1;
    sm.l[warp][g] = l0;
    sm.l[warp][g + 8] = l1;
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int d = 64 * e + 16 * c + t;
      if (g < nr) {
        sm.o[warp][g][d] = o[e * 8 + t][0];
        sm.o[warp][g][d + 8] = o[e * 8 + t][1];
      }
      if (g + 8 < nr) {
        sm.o[warp][g + 8][d] = o[e * 8 + t][2];
        sm.o[warp][g + 8][d + 8] = o[e * 8 + t][3];
      }
    }
  __syncthreads();
  for (int i = tid; i < nr * D; i += kFewWarps * 32) {
    const int r = i / D, d = i - r * D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, sm.m[w][r]);
    const float U = M == -INFINITY ? 0.0f : M;
    float acc = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float f = fast_exp2(sm.m[w][r] - U);
      acc = fmaf(f, sm.o[w][r][d], acc);
      L = fmaf(f, sm.l[w][r], L);
    }
    sm.co[r][d] = acc;
    if (d == 0) {
      sm.cm[r] = M;
      sm.cl[r] = L;
    }
  }
  // ---- join the CTAs: each takes its share of the columns ----
  if (X > 1)
    cluster_barrier();
  else
    __syncthreads();
  const int cols = D / X;
  for (int i = tid; i < nr * cols / 2; i += kFewWarps * 32) {
    const int r = i / (cols / 2), d = rank * cols + (i - r * (cols / 2)) * 2;
    float M = -INFINITY;
    for (int x = 0; x < X; ++x) M = fmaxf(M, ld_peer(&sm.cm[r], x));
    const float U = M == -INFINITY ? 0.0f : M;
    float y0 = 0.0f, y1 = 0.0f, L = 0.0f;
    for (int x = 0; x < X; ++x) {
      const float f = fast_exp2(ld_peer(&sm.cm[r], x) - U);
      y0 = fmaf(f, ld_peer(&sm.co[r][d], x), y0);
      y1 = fmaf(f, ld_peer(&sm.co[r][d + 1], x), y1);
      L = fmaf(f, ld_peer(&sm.cl[r], x), L);
    }
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
    uint16_t* dst = a.out + (int64_t(ch) * a.rows_per_chunk + r0 + r) * a.o_rs +
                    int64_t(h) * a.o_hs + d;
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(y0 * inv, y1 * inv);
  }
  if (X > 1) cluster_barrier();  // no CTA leaves while another reads its memory
}

// ---------------------------------------------------------------------------
// Attention of 128-row tiles on tcgen05
// ---------------------------------------------------------------------------
// One CTA a (segment, group); a step is one listed half block of 64 keys.  Two
// K and two V buffers, two S buffers of 64 columns in TMEM (P overwrites its S
// as bf16 pairs) and O: 256 columns, so two CTAs share an SM.  Warp 0 loads
// (TMA), warp 1 issues the MMAs in the order
//   QK(0) QK(1) | PV(0) QK(2) | PV(1) QK(3) | ...
// and warps 2-5 are the softmax (thread = row = TMEM lane).  S(j+1) is ready
// while the softmax of step j runs.
//   The tensor pipe runs a CTA's MMAs in issue order: QK(j+2), which overwrites
// P(j), follows PV(j).  PV(j) runs during the softmax of j + 1, so a row whose
// maximum grew waits for PV(j) before it rescales O.
//   K buffer j & 1 is free once S(j) has committed, V buffer j & 1 once PV(j)
// has: their next loads have a step and a half to arrive in.
//   Rows of V behind a segment's end are zeroed in shared memory: their weights
// are 0, but 0 * inf would not be.
//   What bounds it: neither pipe by itself.  468 tiles of 32 steps on 296 places (two
// waves, the second 58% full) take 77 us, about 2200 cycles a step of an SM's two
// CTAs.  Their MMAs take 1280 of these (one of N = 64 takes 48 cycles, bound by
// shared memory, one of N = 128 64; 16 and 8 of them a step), the softmax of a CTA
// alone on its SM 1030 (clock64, D = 64: 96 for the scores, 826 for maxima and
// weights, 100 to store and signal); the rest is the way from one role to the next.
// Issued by lane 0 instead of an elected lane an MMA of N = 64 takes 55 to 66 cycles:
// 36 segments (468 tiles) took 144.6 us with their means and selection instead of
// 141.4, 144 segments 507 instead of 495.
//   Groups of 17 to 64 rows take a tile of 128 all the same: half of every MMA and
// two of the four softmax warps have nothing to do then.
//   Not kept, the first ones in separate runs, which differ by up to 3%: 128-key
// steps with one S buffer 89 to 92 us against 82 for the 468 tiles; Q.K of 128 keys
// with the softmax and P.V in halves 93; the next keys pulled into L2 86; a third K
// buffer 81; a row's columns split over two warps 143.5 against 139.5 (in turn, with
// means and selection).
constexpr int kTcThreads = 192;
constexpr int kStepKeys = 64;
constexpr int kMaxHalves = 2 * kMaxTopK;

template <int D>
struct __align__(1024) SparseTcSmem {
  uint8_t q[kBM * D * 2];
  uint8_t k[2][kStepKeys * D * 2];
  uint8_t v[2][kStepKeys * D * 2];
  uint64_t q_full, k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2], drain;
  uint32_t tmem_base;
  int abort, halves;
  int list[kMaxHalves];
};

// Row max over 64 raw scores held as bits.
__device__ __forceinline__ float row_max64(const uint32_t (&s)[2][32]) {
  float m[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float a[11];
#pragma unroll
    for (int i = 0; i < 10; ++i)
      a[i] = max3(__uint_as_float(s[q][3 * i]), __uint_as_float(s[q][3 * i + 1]),
                  __uint_as_float(s[q][3 * i + 2]));
    a[10] = fmaxf(__uint_as_float(s[q][30]), __uint_as_float(s[q][31]));
    const float b0 = max3(a[0], a[1], a[2]), b1 = max3(a[3], a[4], a[5]);
    const float b2 = max3(a[6], a[7], a[8]), b3 = fmaxf(a[9], a[10]);
    m[q] = fmaxf(max3(b0, b1, b2), b3);
  }
  return fmaxf(m[0], m[1]);
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 2)
    sparse_tc_kernel(const __grid_constant__ CUtensorMap tm_q,
                     const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, SparseArgs a) {
  extern __shared__ uint8_t smem_raw[];
  SparseTcSmem<D>& sm = *reinterpret_cast<SparseTcSmem<D>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kCols = D / 64;                    // 64-column halves of a row
  constexpr uint32_t kQCol = kBM * 64 * 2;         // one of them, 128 query rows
  constexpr uint32_t kKCol = kStepKeys * 64 * 2;   // one of them, 64 keys
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;
  const int unit = blockIdx.x;
  const int s = unit / a.groups, grp = unit - s * a.groups;
  const int ch = s / a.H, h = s - ch * a.H;
  const int r0 = grp * a.query_block;
  const int nr = min(a.query_block, a.rows_per_chunk - r0);

  if (threadIdx.x == 0) {
    sm.abort = 0;
    mbar_init(&sm.q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.pv_done[i], 1);
    }
    mbar_init(&sm.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     su32(&sm.tmem_base)),
                 "r"(256));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  grid_wait();
  const SegView sg = segment(a.cu, s, a.kv_rows);
  if (warp == 1) {  // the listed 64-key halves that hold keys, in order
    const int nblk = (sg.len + a.block - 1) / a.block, per = a.block / 64;
    const int32_t* lst = a.blocks + int64_t(unit) * a.top_k;
    int n = 0;
    for (int b = 0; b < a.top_k; b += 32) {
      const int e = b + lane < a.top_k ? lst[b + lane] : -1;
      int mine = e >= 0 && e < nblk ? per : 0;
      if (mine == 2 && int64_t(e) * 128 + 64 >= sg.len) mine = 1;
      int at = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += y;
      }
      const int total = __shfl_sync(0xffffffffu, at, 31);
      at += n - mine;
      for (int i = 0; i < mine; ++i) sm.list[at + i] = e * per + i;
      n += total;
    }
    if (lane == 0) sm.halves = n;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;  // S0 | S1 | O: 64 + 64 + D columns
  const int steps = sm.halves;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one() && steps > 0) {
      mbar_expect_tx(&sm.q_full, kBM * D * 2);
      const int row0 = ch * a.rows_per_chunk + r0;
#pragma unroll
      for (int x = 0; x < kCols; ++x)
        tma_load_3d(sm.q + x * kQCol, &tm_q, &sm.q_full, 64 * x, h, row0);
      int kj = 0, vj = 0;  // loads issued
      for (int j = 0; j < steps; ++j) {
        const int b = j & 1;
        const uint32_t prev = ((j >> 1) + 1) & 1;  // parity of step j - 2
        const int y = sg.start + sm.list[j] * kStepKeys;
        if (j > 1 && !mbar_wait(&sm.s_full[b], prev, abort, a.status)) break;
        mbar_expect_tx(&sm.k_full[b], kKCol * kCols);
#pragma unroll
        for (int x = 0; x < kCols; ++x)
          tma_load_2d(sm.k[b] + x * kKCol, &tm_k, &sm.k_full[b], 64 * x, y);
        ++kj;
        if (j > 1 && !mbar_wait(&sm.pv_done[b], prev, abort, a.status)) break;
        mbar_expect_tx(&sm.v_full[b], kKCol * kCols);
#pragma unroll
        for (int x = 0; x < kCols; ++x)
          tma_load_2d(sm.v[b] + x * kKCol, &tm_v, &sm.v_full[b], 64 * x, y);
        ++vj;
      }
      if (*abort) {  // this CTA's own copies land before its memory goes away
        const uint64_t t0 = now_ns();
        while (!mbar_try(&sm.q_full, 0) && now_ns() - t0 < kTimeoutNs) {
        }
        for (int j = kj > 2 ? kj - 2 : 0; j < kj; ++j)
          while (!mbar_try(&sm.k_full[j & 1], (j >> 1) & 1) && now_ns() - t0 < kTimeoutNs) {
          }
        for (int j = vj > 2 ? vj - 2 : 0; j < vj; ++j)
          while (!mbar_try(&sm.v_full[j & 1], (j >> 1) & 1) && now_ns() - t0 < kTimeoutNs) {
          }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one() && steps > 0) {
      constexpr uint32_t kN = uint32_t(kBN >> 3) << 17;  // N of idesc_bf16
      constexpr uint32_t id_qk = (idesc_bf16(false) & ~kN) | (uint32_t(kStepKeys >> 3) << 17);
      constexpr uint32_t id_pv = (idesc_bf16(true) & ~kN) | (uint32_t(D >> 3) << 17);
      const uint64_t dq = sdesc_sw128(su32(sm.q), 16, 1024);
      const uint64_t dv = sdesc_sw128(su32(sm.v[0]), kKCol, 1024);
      const uint32_t d_hi = uint32_t(dq >> 32), v_hi = uint32_t(dv >> 32);
      const uint32_t q_lo = uint32_t(dq), v_lo0 = uint32_t(dv);
      const uint32_t v_lo1 = uint32_t(sdesc_sw128(su32(sm.v[1]), kKCol, 1024));
      const uint32_t k_lo0 = uint32_t(sdesc_sw128(su32(sm.k[0]), 16, 1024));
      const uint32_t k_lo1 = uint32_t(sdesc_sw128(su32(sm.k[1]), 16, 1024));
      auto issue_qk = [&](int b) {
        const uint32_t k_lo = b ? k_lo1 : k_lo0;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qo = ((kk >> 2) * kQCol + (kk & 3) * 32) >> 4;
          const uint32_t ko = ((kk >> 2) * kKCol + (kk & 3) * 32) >> 4;
          mma_ss(tmem + b * 64, (uint64_t(d_hi) << 32) | (q_lo + qo),
                 (uint64_t(d_hi) << 32) | (k_lo + ko), id_qk, kk > 0 ? 1u : 0u);
        }
        tc_commit(&sm.s_full[b]);
      };
      bool ok = mbar_wait(&sm.q_full, 0, abort, a.status);
      for (int j = 0; ok && j < 2 && j < steps; ++j) {
        ok = mbar_wait(&sm.k_full[j], 0, abort, a.status);
        if (!ok) break;
        tc_fence_after();
        issue_qk(j);
      }
      for (int j = 0; ok && j < steps; ++j) {
        const int b = j & 1;
        const uint32_t par = (j >> 1) & 1;
        ok = mbar_wait(&sm.v_full[b], par, abort, a.status) &&
             mbar_wait(&sm.p_full[b], par, abort, a.status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_lo = b ? v_lo1 : v_lo0;
#pragma unroll
        for (int kk = 0; kk < kStepKeys / 16; ++kk)
          mma_ts(tmem + 128, tmem + b * 64 + kk * 8,
                 (uint64_t(v_hi) << 32) | (v_lo + ((kk * 2048) >> 4)), id_pv,
                 (kk > 0 || j > 0) ? 1u : 0u);
        tc_commit(&sm.pv_done[b]);
        if (j + 2 < steps) {
          ok = mbar_wait(&sm.k_full[b], par ^ 1, abort, a.status);
          if (!ok) break;
          tc_fence_after();
          issue_qk(b);
        }
      }
      // every MMA issued here completes before the CTA frees TMEM
      tc_commit(&sm.drain);
      const uint64_t t0 = now_ns();
      while (!mbar_try(&sm.drain, 0) && now_ns() - t0 < kTimeoutNs) {
      }
    }
  } else {
    // ---------------- softmax, correction, output ----------------
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    const uint32_t o_tm = tmem + 128 + lane_off;
    const float sc = a.scale_log2;
    // A lane whose wait ran out waits no more but stays with its warp to the end
    // (its warp's votes and TMEM accesses need every lane): what it reads and writes
    // is this CTA's own memory, and no row is stored.
    float m_ref = -INFINITY, l_sum = 0.0f;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int b = j & 1;
      const uint32_t par = (j >> 1) & 1;
      const uint32_t s_tm = tmem + b * 64 + lane_off;
      const int valid = sg.len - sm.list[j] * kStepKeys;  // keys inside the segment
      const bool partial = valid < kStepKeys;
      ok = ok && mbar_wait(&sm.s_full[b], par, abort, a.status);
      tc_fence_after();
      if (partial) {
        ok = ok && mbar_wait(&sm.v_full[b], par, abort, a.status);
        if (row < kStepKeys && row >= valid) {  // this row of V holds no key
#pragma unroll
          for (int x = 0; x < kCols; ++x)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(sm.v[b] + x * kKCol + row * 128 + e * 16) =
                  make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
      }
      if (quad * 32 >= nr) {  // no row of this warp is the group's: P and O may
        __syncwarp();         // hold anything there
        if (lane == 0) mbar_arrive(&sm.p_full[b]);
        continue;
      }
      uint32_t sr[2][32];
      tmem_ld32(s_tm, sr[0]);
      tmem_ld32(s_tm + 32, sr[1]);
      tmem_wait_ld();
      if (partial) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (q * 32 + e >= valid) sr[q][e] = __float_as_uint(-INFINITY);
      }
      const float m_new = fmaxf(m_ref, row_max64(sr) * sc);
      const bool grow = m_new > m_ref + kRescaleThreshold || j == 0;
      float alpha = 1.0f;
      if (grow) {
        alpha = (j == 0 || m_ref == -INFINITY) ? 0.0f : fast_exp2(m_ref - m_new);
        m_ref = m_new;
      }
      // a row whose scores are all -inf keeps a reference of 0; one of +inf (a finite
      // score that overflows when scaled too) makes the row NaN: inf * 0
      const float m_use = m_ref == -INFINITY ? 0.0f : fmaf(m_ref, 0.0f, m_ref);
      const f2 scale2 = mk2(sc, sc), negm2 = mk2(-m_use, -m_use);
      f2 acc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = mk2(0.0f, 0.0f);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t pr[16];
        if (partial)
          softmax_chunk<false>(sr[q], scale2, negm2, acc[2 * q], acc[2 * q + 1], pr);
        else
          softmax_chunk<true>(sr[q], scale2, negm2, acc[2 * q], acc[2 * q + 1], pr);
        tmem_st16(s_tm + q * 16, pr);
      }
      acc[0] = add2(add2(acc[0], acc[1]), add2(acc[2], acc[3]));
      float e0, e1;
      un2(acc[0], e0, e1);
      l_sum = l_sum * alpha + (e0 + e1);
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        // PV(j - 1) may still be running
        ok = ok && mbar_wait(&sm.pv_done[b ^ 1], ((j - 1) >> 1) & 1, abort, a.status);
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t orr[32];
          tmem_ld32(o_tm + q * 32, orr);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) orr[e] = __float_as_uint(__uint_as_float(orr[e]) * alpha);
          tmem_st32(o_tm + q * 32, orr);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[b]);
    }
    uint16_t* dst = a.out + (int64_t(ch) * a.rows_per_chunk + r0 + row) * a.o_rs +
                    int64_t(h) * a.o_hs;
    if (steps == 0) {
      if (row < nr)
        for (int e = 0; e < D; e += 8)
          *reinterpret_cast<uint4*>(dst + e) = make_uint4(0, 0, 0, 0);
    } else if (__all_sync(0xffffffffu,
                          ok && mbar_wait(&sm.pv_done[(steps - 1) & 1], ((steps - 1) >> 1) & 1,
                                          abort, a.status))) {
      tc_fence_after();
      const float inv = l_sum > 0.0f ? 1.0f / l_sum : (l_sum == 0.0f ? 0.0f : l_sum);
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        uint32_t orr[32];
        tmem_ld32(o_tm + q * 32, orr);
        tmem_wait_ld();
        if (row < nr) store_row32(dst + q * 32, orr, inv);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
bool shape_ok(int num_chunks, int H, int rows_per_chunk, int query_block, int block, int top_k) {
  return num_chunks >= 0 && H >= 0 && rows_per_chunk >= 0 && query_block >= 1 &&
         query_block <= kBM && (block == 64 || block == 128) && top_k >= 1;
}

// One-dimensional grid of units in clusters of X.
template <typename A>
int launch_units(void (*kernel)(A), const A& a, int64_t units, int X, bool early, int threads,
                 size_t smem, cudaStream_t stream) {
  if (units * X >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  return launch_clusters(kernel, dim3(unsigned(units * X)), X, early, threads, smem, stream, a);
}

template <int D, int X>
int select_shape(const SelectArgs& a, int64_t units, cudaStream_t stream) {
  static std::mutex mu;
  static int done[kMaxDevices] = {};
  if (smem_opt_in(done, mu, select_blocks_kernel<D, X>, select_bytes(D, X, kMaxTopK)) <= 0) {
    cudaGetLastError();
    return PKV_ELAUNCH;
  }
  return launch_units(select_blocks_kernel<D, X>, a, units, X, true, kSelThreads,
                      select_bytes(D, X, a.top_k), stream);
}

template <int D>
int select_few(const SelectArgs& a, int64_t groups, cudaStream_t stream) {
  static std::mutex mu;
  static int done[kMaxDevices] = {};
  const auto bytes = [](int top_k) { return sizeof(GroupSmem) + size_t(top_k + kSelChunk) * 12; };
  if (smem_opt_in(done, mu, select_group_kernel<D>, bytes(kMaxTopK)) <= 0) {
    cudaGetLastError();
    return PKV_ELAUNCH;
  }
  // a cluster while the groups leave SMs idle and the keys could make blocks
  // enough to share (16 a round and CTA)
  int X = 1;
  while (X < kSelCluster && groups * X * 2 <= sm_count() && a.kv_rows / a.block >= int64_t(X) * 64)
    X *= 2;
  return launch_units(select_group_kernel<D>, a, groups, X, true, kSelThreads, bytes(a.top_k),
                      stream);
}

// The form by what a group costs.  select_group_kernel reads the whole table
// for every group; select_blocks_kernel reads it once for 16, but an mma has 16
// rows however few groups a segment has.  Measured, us with D = 128 (group form
// / tensor cores): one group a segment 9.4 / 12.5 (12 x 512 blocks), 43 / 87
// (400 x 512), 100 / 148 (20 x 7812); 16 groups a segment 9.8 / 13.8 (8 x 128
// blocks), 13.0 / 13.9 (8 x 256), 14.6 / 14.0 (4 x 512), 15.3 / 13.7 (8 x 300),
// 19.7 / 13.9 (8 x 512).  With more than one group they meet at about 220 blocks an
// SM in all.  (Not so for a few very long segments: 4 x 13 groups of 4000 blocks take
// 75 / 102 and go to the tensor cores all the same.)
// On the tensor cores, eight CTAs a cluster where that leaves room for all of
// them at once (a cluster shares a few SMs of one GPC, so not every SM can be
// used; 14.2 us against 16.0 with four for 12 x 13 groups of 437 blocks), else four
// (19.6 against 26.1 with eight for 36 x 13 groups of 300).
template <int D>
int launch_select(SelectArgs a, int64_t segs, cudaStream_t stream) {
  const int64_t blocks = a.kv_rows / a.block + segs;  // of all segments, at most
  if (a.groups == 1 || a.groups * blocks <= int64_t(220) * sm_count())
    return select_few<D>(a, segs * a.groups, stream);
  a.packs = (a.groups + kSelGroups - 1) / kSelGroups;
  const int64_t units = segs * a.packs;
  if (units * 8 <= sm_count()) return select_shape<D, 8>(a, units, stream);
  return select_shape<D, 4>(a, units, stream);
}

template <int D>
int launch_few(const SparseArgs& a, int64_t units, cudaStream_t stream) {
  static std::mutex mu;
  static int done[kMaxDevices] = {};
  const size_t smem = sizeof(FewSmem<D>);
  if (smem_opt_in(done, mu, sparse_few_kernel<D>, smem) <= 0) {
    cudaGetLastError();
    return PKV_ELAUNCH;
  }
  // the cluster: a warp gets a chunk at least, and the grid stays within a
  // few CTAs an SM
  const int chunks = a.top_k * (a.block / 16);
  int X = 1;
  while (X < 8 && X * kFewWarps < chunks && units * X < int64_t(sm_count()) * 2) X *= 2;
  return launch_units(sparse_few_kernel<D>, a, units, X, true, kFewWarps * 32, smem, stream);
}

template <int D>
int launch_tc(const SparseArgs& a, int num_chunks, int64_t units, cudaStream_t stream) {
  CUtensorMap mq, mk, mv;
  // (no keys at all: every list is empty and no K/V tile is loaded; the maps
  // then only have to be well formed)
  const void* kb = a.kv_rows > 0 ? a.k : a.q;
  const void* vb = a.kv_rows > 0 ? a.v : a.q;
  const cuuint64_t kv_dims[2] = {cuuint64_t(D), cuuint64_t(a.kv_rows > 0 ? a.kv_rows : 1)};
  const cuuint64_t kv_str[1] = {cuuint64_t(D) * 2};
  const cuuint32_t kv_box[2] = {64, 64};
  const cuuint64_t q_dims[3] = {cuuint64_t(D), cuuint64_t(a.H),
                                cuuint64_t(num_chunks) * a.rows_per_chunk};
  const cuuint64_t q_str[2] = {cuuint64_t(a.q_hs > 0 ? a.q_hs : D) * 2, cuuint64_t(a.q_rs) * 2};
  const cuuint32_t q_box[3] = {64, 1, kBM};
  if (!make_map(&mk, kb, 2, kv_dims, kv_str, kv_box) ||
      !make_map(&mv, vb, 2, kv_dims, kv_str, kv_box) ||
      !make_map(&mq, a.q, 3, q_dims, q_str, q_box))
    return PKV_EUNSUPPORTED;
  // at least 100 KB, so that no third CTA comes to an SM (TMEM holds two)
  size_t smem = sizeof(SparseTcSmem<D>) + 1024;
  if (smem < 100 * 1024) smem = 100 * 1024;
  static std::mutex mu;
  static int done[kMaxDevices] = {};
  if (smem_opt_in(done, mu, sparse_tc_kernel<D>, smem) <= 0) {
    cudaGetLastError();
    return PKV_ELAUNCH;
  }
  // (early: 30.9 -> 29.9 us for 112 tiles of 16 steps with their selection and
  // means, 146.4 -> 145.2 for 468)
  return launch_clusters(sparse_tc_kernel<D>, dim3(unsigned(units)), 1, true, kTcThreads, smem,
                         stream, mq, mk, mv, a);
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_block_rows(int64_t kv_rows, int segments, int block) {
  if (kv_rows < 0 || segments < 0 || (block != 64 && block != 128)) return 0;
  return kv_rows / block + segments;
}

extern "C" int pkv_block_means(const uint16_t* k, int64_t kv_rows, int head_dim,
                               const int32_t* cu_seqlens_k, int segments, int block, float* means,
                               int64_t means_rows, int zero_rest, pkv_stream_t stream) {
  if (kv_rows < 0 || segments < 0 || means_rows < 0 || (block != 64 && block != 128))
    return PKV_EINVAL;
  if (segments == 0 || means_rows == 0) return PKV_OK;
  if ((kv_rows > 0 && !k) || !cu_seqlens_k || !means) return PKV_EINVAL;
  if ((head_dim != 64 && head_dim != 128) || kv_rows >= (int64_t(1) << 31) ||
      reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(means) % 16)
    return PKV_EUNSUPPORTED;
  // four warps a row while one would not fill the GPU: 246 blocks of 128 keys
  // of 64 take 5 us instead of 8
  const bool few = means_rows <= int64_t(sm_count()) * 8;
  int64_t grid = few ? (means_rows + 1) / 2 : (means_rows + 7) / 8;
  const int64_t cap = int64_t(sm_count()) * 8;
  if (grid > cap) grid = cap;
  auto s = static_cast<cudaStream_t>(stream);
  auto kernel = head_dim == 128 ? (few ? block_means_kernel<128, 4> : block_means_kernel<128, 1>)
                                : (few ? block_means_kernel<64, 4> : block_means_kernel<64, 1>);
  kernel<<<int(grid), 256, 0, s>>>(k, kv_rows, cu_seqlens_k, segments, block, means, means_rows,
                                   zero_rest);
  return launch_status();
}

extern "C" int pkv_select_blocks(const uint16_t* q, int64_t q_row_stride, int64_t q_head_stride,
                                 const float* means, int64_t means_rows,
                                 const int32_t* cu_seqlens_k, int64_t kv_rows, int num_chunks,
                                 int num_heads, int rows_per_chunk, int head_dim, int query_block,
                                 int block, int top_k, int32_t* blocks, pkv_stream_t stream) {
  if (!shape_ok(num_chunks, num_heads, rows_per_chunk, query_block, block, top_k) ||
      means_rows < 0 || kv_rows < 0)
    return PKV_EINVAL;
  if (num_chunks == 0 || num_heads == 0 || rows_per_chunk == 0) return PKV_OK;
  if (!q || (means_rows > 0 && !means) || !cu_seqlens_k || !blocks) return PKV_EINVAL;
  if (top_k > kMaxTopK) return PKV_ECAPACITY;
  if ((head_dim != 64 && head_dim != 128) || kv_rows >= (int64_t(1) << 31) ||
      int64_t(num_chunks) * rows_per_chunk >= (int64_t(1) << 31) - kBM ||
      reinterpret_cast<uintptr_t>(q) % 16 || q_row_stride % 8 || q_head_stride % 8 || reinterpret_cast<uintptr_t>(means) % 16)
    return PKV_EUNSUPPORTED;
  SelectArgs a{};
  a.q = q;
  a.q_rs = q_row_stride;
  a.q_hs = q_head_stride;
  a.kv_rows = kv_rows;
  a.means_rows = means_rows;
  a.means = means;
  a.cu = cu_seqlens_k;
  a.blocks = blocks;
  a.H = num_heads;
  a.rows_per_chunk = rows_per_chunk;
  a.groups = (rows_per_chunk + query_block - 1) / query_block;
  a.query_block = query_block;
  a.block = block;
  a.top_k = top_k;
  const int64_t segs = int64_t(num_chunks) * num_heads;
  if (segs * a.groups >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  auto s = static_cast<cudaStream_t>(stream);
  return head_dim == 128 ? launch_select<128>(a, segs, s) : launch_select<64>(a, segs, s);
}

extern "C" int pkv_block_attention(const uint16_t* q, int64_t q_row_stride, int64_t q_head_stride,
                                   const uint16_t* k, const uint16_t* v, int64_t kv_rows,
                                   const int32_t* cu_seqlens_k, int num_chunks, int num_heads,
                                   int rows_per_chunk, int head_dim, float softmax_scale,
                                   const int32_t* blocks, int query_block, int block, int top_k,
                                   uint16_t* out, int64_t o_row_stride, int64_t o_head_stride,
                                   int32_t* status, pkv_stream_t stream) {
  if (!shape_ok(num_chunks, num_heads, rows_per_chunk, query_block, block, top_k) || kv_rows < 0)
    return PKV_EINVAL;
  if (num_chunks == 0 || num_heads == 0 || rows_per_chunk == 0) return PKV_OK;
  if (!q || (kv_rows > 0 && (!k || !v)) || !cu_seqlens_k || !blocks || !out) return PKV_EINVAL;
  if (!(softmax_scale > 0.0f)) return PKV_EINVAL;
  if (top_k > kMaxTopK) return PKV_ECAPACITY;
  const int64_t q_rows = int64_t(num_chunks) * rows_per_chunk;
  if ((head_dim != 64 && head_dim != 128) || kv_rows >= (int64_t(1) << 31) ||
      q_rows >= (int64_t(1) << 31) - kBM || reinterpret_cast<uintptr_t>(q) % 16 ||
      reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16 ||
      reinterpret_cast<uintptr_t>(out) % 16 || q_row_stride % 8 || q_head_stride % 8 ||
      o_row_stride % 8 || o_head_stride % 8 || q_row_stride <= 0 ||
      (q_head_stride <= 0 && num_heads > 1))
    return PKV_EUNSUPPORTED;
  SparseArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_rs = q_row_stride;
  a.q_hs = q_head_stride;
  a.kv_rows = kv_rows;
  a.o_rs = o_row_stride;
  a.o_hs = o_head_stride;
  a.cu = cu_seqlens_k;
  a.blocks = blocks;
  a.out = out;
  a.status = status;
  a.H = num_heads;
  a.rows_per_chunk = rows_per_chunk;
  a.groups = (rows_per_chunk + query_block - 1) / query_block;
  a.query_block = query_block;
  a.block = block;
  a.top_k = top_k;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  const int64_t units = int64_t(num_chunks) * num_heads * a.groups;
  if (units >= (int64_t(1) << 31)) return PKV_EUNSUPPORTED;
  auto s = static_cast<cudaStream_t>(stream);
  const int rows = query_block < rows_per_chunk ? query_block : rows_per_chunk;
  if (rows <= kFewRows)
    return head_dim == 128 ? launch_few<128>(a, units, s) : launch_few<64>(a, units, s);
  return head_dim == 128 ? launch_tc<128>(a, num_chunks, units, s)
                         : launch_tc<64>(a, num_chunks, units, s);
}
