// Acceptance of drafted tokens by the residual rule, from given uniform
// numbers: the output is distributed as the target's own samples whatever the
// draft proposed.  (verify_new, diffspec/draft/tree_verification.py:100-162,
// samples one token per node and matches drafts against it; this is the rule
// of speculative sampling.)
//
// At a node with target distribution p the children are tried in index order:
//   fixed drafts (no draft probabilities): child x is accepted when
//     u * (1 - removed) < p(x); a rejected x leaves the distribution
//     (removed += p(x); a second child with the same token is never accepted);
//   sampled drafts, each child drawn from the node's draft distribution q:
//     after k rejections the distribution is (p - a q)+ / b with a = 0, b = 1
//     at first, and a += b, b = sum (p - a q)+ after a rejection, because
//     ((p - a q)+ / b - q)+ = (p - (a + b) q)+ / b; child x is accepted when
//     u * b * q(x) < (p(x) - a q(x))+.
// The walk goes on at the accepted child; where none is accepted the next
// token is drawn from what is left of the distribution by inverting its CDF.
//
// Stage 1 (grid chunks x nodes x batch) reads every node's logits once and
// leaves a (max, sum) pair per chunk: bound by HBM.  Stage 2 (one cluster per
// sequence) joins the pairs, walks the tree, and draws: the ending node's row
// is split over the cluster's CTAs, whose sums meet through distributed
// shared memory.
//
// Whole numbers hang on comparisons here.  A draw goes wrong when uniform[0]
// falls between a border of the exact CDF and the computed one, and 128256
// words have as many borders: with fp32 weights (2^-24 each) that is a few
// draws in ten thousand.  Stage 2 therefore carries weights and sums as
// unevaluated pairs of floats (about 2^-36 a weight, one draw in a million);
// FP64 instructions would do too, but run at 1/24 of the fp32 rate here (49 us
// for one row of 128256 words on eight SMs; the pairs take 4 on sixteen).
// Stage 1's normaliser (fp32 exponentials, summed in 64 bits) enters only the
// few comparisons of a child's probability.
//
// A tree of 65 over 128256 words takes 18.0 us: about 6 for stage 1 (2.5 at the
// measured HBM rate), then 2 to join the pairs, 2 for the walk, 4 for the pass
// over the ending row, 2 for the draw, each a few dependent round trips.  32
// sampled trees of 9 take 62 us, stage 1 19 of them (11.3 at the HBM rate): a pass
// over 32064 words an SM is 9 us of issue (some 65 instructions a word), and the
// sequence with the most rejections makes three or four.
#include <cooperative_groups.h>

#include <atomic>
#include <cmath>

#include "common.cuh"

namespace tv {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256;
constexpr int kChunkBytes = 16384;      // logits per stage-1 CTA: four 16-byte loads a thread
constexpr int kWalkThreads = 512;
constexpr int kWalkWarps = kWalkThreads / 32;
constexpr int kMaxCluster = 16;

template <typename E> __device__ __forceinline__ float as_float(E x);
template <> __device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float as_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float as_float<float>(float x) { return x; }

// ---- pairs of floats: h + l, |l| at most half a step of h (Dekker; Knuth) -----
struct Pair {
  float h, l;
};
__device__ __forceinline__ Pair two_sum(float a, float b) {
  const float s = a + b, bb = s - a;
  return {s, (a - (s - bb)) + (b - bb)};
}
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  const Pair s = two_sum(a.h, b.h);
  const float l = s.l + (a.l + b.l);
  const float h = s.h + l;
  return {h, l - (h - s.h)};
}
__device__ __forceinline__ double value(Pair a) { return (double)a.h + (double)a.l; }
__device__ __forceinline__ Pair pair_of(double d) {
  const float h = (float)d;
  return {h, (float)(d - (double)h)};
}
__device__ __forceinline__ Pair warp_sum(Pair a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = add(a, {__shfl_xor_sync(0xffffffffu, a.h, o), __shfl_xor_sync(0xffffffffu, a.l, o)});
  return a;
}

constexpr int kTable = 1024;     // 2^(i / 1024) as pairs

// Maximum that keeps a NaN of either side.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// How exponents become weights: 1024 log2(e) / T as a pair, and the smallest
// l - m that is told from -inf (2^-200).
struct Exponent {
  Pair c;
  float floor;
};

// exp((l - m) / T): t = (l - m) * 1024 log2(e) / T as a pair, its nearest
// integer (by adding 1.5 * 2^23) splits into a power of two and a table entry,
// and the rest r (at most 1/2) is 2^(r / 1024) = 1 + y + y^2 / 2 + y^3 / 6 with
// y < 3.4e-4.  Below 2^-126 of the largest weight: 0.  The low part is up to
// 3.4e-4 of the high one, no unevaluated rounding error, until it is summed.
// l - m of 16-bit logits is exact or, for |l| below 2^-13 of m, off by 2^-24
// of m at most; fp32 logits carry the difference's error along (EXACT).
template <bool EXACT>
__device__ __forceinline__ Pair weight_pair(float l, float m, const Exponent& c, const float2* table) {
  float x, xl = 0.f;
  if (EXACT) {
    const Pair d = two_sum(l, -m);
    x = max_nan(d.h, c.floor);
    xl = x == d.h ? d.l : 0.f;
  } else {
    x = max_nan(l - m, c.floor);
  }
  const float t = x * c.c.h;
  float tl = fmaf(x, c.c.l, fmaf(x, c.c.h, -t));
  if (EXACT) tl = fmaf(xl, c.c.h, tl);
  const float kf = t + 12582912.0f;
  const float y = ((t - (kf - 12582912.0f)) + tl) * 6.7690154351557159e-4f;   // ln(2) / 1024
  const int ki = __float_as_int(kf) - 0x4B400000;
  const float2 e = table[ki & (kTable - 1)];
  const float s = fmaf(y * y, fmaf(y, 1.0f / 6.0f, 0.5f), y);
  const float scale = __int_as_float((max(ki >> 10, -127) + 127) << 23);
  return {e.x * scale, fmaf(e.x, s, e.y) * scale};
}

struct Args {
  const void* logits;
  int64_t l_sb, l_sm;
  int rows, vocab, chunk, chunks;
  int blocks;                  // 256-word blocks per CTA of a stage-2 cluster
  const int64_t* draft;
  int64_t d_sb;
  const int64_t* parent;
  int64_t p_sb;
  const int32_t* counts;
  const float* uniform;
  int64_t u_sb;
  const void* probs;
  int64_t q_sb, q_sm;
  float c_hi, c_lo;            // log2(e) / T as a sum of two floats, c_lo > 0
  Exponent exponent;
  float* part_max;             // [batch][rows][chunks]
  double* part_sum;
  int64_t* next_tokens;        // [batch][rows]
  int64_t* result;             // [batch][8 + 2 rows]
};

// exp((l - m) / T) in fp32.  Of the rounding errors only the product's own
// stays, one of either sign a word; c_lo takes out that of log2(e) / T, which
// all words share (and is positive, so that -inf stays -inf).
__device__ __forceinline__ float weight32(float l, float m, float c_hi, float c_lo) {
  const float x = l - m;
  return fast_exp2(fmaf(x, c_lo, x * c_hi));
}

template <typename E>
__global__ void __launch_bounds__(kStatThreads) row_stats_kernel(const Args a) {
  constexpr int VEC = 16 / sizeof(E);
  constexpr int U = kChunkBytes / (16 * kStatThreads);
  grid_wait();
  grid_next();        // not before: stage 2 reads its inputs ahead of its own wait
  const int row = blockIdx.y, b = blockIdx.z;
  if (a.counts && row >= a.counts[b]) return;
  const int lo = blockIdx.x * a.chunk;
  const int hi = min(a.vocab, lo + a.chunk);
  const E* src = static_cast<const E*>(a.logits) + (int64_t)b * a.l_sb + (int64_t)row * a.l_sm;
  // elements before the first 16-byte boundary and after the last go one by one
  const int head = min(hi - lo, (int)(((16 - (reinterpret_cast<uintptr_t>(src + lo) & 15)) & 15) / sizeof(E)));
  const int nvec = (hi - lo - head) / VEC;
  const uint4* vsrc = reinterpret_cast<const uint4*>(src + lo + head);
  const int tail = lo + head + nvec * VEC;
  uint4 raw[U];
  float one[2];
  int n1 = 0;
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (threadIdx.x + i * kStatThreads < nvec) raw[i] = vsrc[threadIdx.x + i * kStatThreads];
  if ((int)threadIdx.x < head) one[n1++] = as_float<E>(src[lo + threadIdx.x]);
  if (tail + (int)threadIdx.x < hi) one[n1++] = as_float<E>(src[tail + threadIdx.x]);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (threadIdx.x + i * kStatThreads < nvec) {
      const E* e = reinterpret_cast<const E*>(&raw[i]);
#pragma unroll
      for (int k = 0; k < VEC; ++k) m = fmaxf(m, as_float<E>(e[k]));
    }
  if (n1 > 0) m = fmaxf(m, one[0]);
  if (n1 > 1) m = fmaxf(m, one[1]);
  __shared__ float wm[kStatThreads / 32];
  __shared__ double ws[kStatThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) wm[warp] = m;
  __syncthreads();
  m = wm[0];
#pragma unroll
  for (int w = 1; w < kStatThreads / 32; ++w) m = fmaxf(m, wm[w]);
  const float base = m == -INFINITY ? 0.f : m;      // a chunk that the mask empties sums to 0
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (threadIdx.x + i * kStatThreads < nvec) {
      const E* e = reinterpret_cast<const E*>(&raw[i]);
#pragma unroll
      for (int k = 0; k < VEC; ++k) s += weight32(as_float<E>(e[k]), base, a.c_hi, a.c_lo);
    }
  if (n1 > 0) s += weight32(one[0], base, a.c_hi, a.c_lo);
  if (n1 > 1) s += weight32(one[1], base, a.c_hi, a.c_lo);
  double d = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if (lane == 0) ws[warp] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kStatThreads / 32; ++w) d += ws[w];
    const int64_t at = ((int64_t)b * a.rows + row) * a.chunks + blockIdx.x;
    a.part_max[at] = m;
    a.part_sum[at] = d;
  }
}

// Words are summed in blocks of 256 (eight a lane, so eight loads are in
// flight); a CTA's blocks are contiguous and their sums stay in shared memory,
// so the draw finds its block without a second pass over the row.
constexpr int kLane = 8;
constexpr int kBlock = 32 * kLane;

struct Walk {
  float2 table[kTable];
  double cta_sum[2][kMaxCluster];
  int status;
  int removed;            // words taken out of the ending node's distribution, in dup[]
};

// Q: type of the draft probabilities (float without any when SAMPLED is false).
template <typename E, typename Q, bool SAMPLED>
__global__ void __launch_bounds__(kWalkThreads, 1) walk_kernel(const Args a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), size = (int)cluster.num_blocks();
  const int b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.rows, vocab = a.vocab;
  __shared__ Walk sh;
  extern __shared__ __align__(16) uint8_t dyn[];
  double* z = reinterpret_cast<double*>(dyn);                 // [rows] normaliser
  double* prob = z + rows;                                     // [rows] p(draft) at the parent
  double* block_sum = prob + rows;                             // [blocks of this CTA]
  int64_t* tok = reinterpret_cast<int64_t*>(block_sum + a.blocks);  // [rows]
  float* mx = reinterpret_cast<float*>(tok + rows);            // [rows] row maximum
  int* par = reinterpret_cast<int*>(mx + rows);                // [rows]
  int* take = par + rows;                                      // [rows] accepted child or -1
  int* dup = take + rows;                                      // [rows] an earlier sibling has the same word
  const int64_t* draft = a.draft + (int64_t)b * a.d_sb;
  const int64_t* parent = a.parent + (int64_t)b * a.p_sb;
  const float* u = a.uniform + (int64_t)b * a.u_sb;
  int64_t* result = a.result + (int64_t)b * (8 + 2 * rows);
  int64_t* next_tokens = a.next_tokens + (int64_t)b * rows;
  const E* logits = static_cast<const E*>(a.logits) + (int64_t)b * a.l_sb;
  for (int i = tid; i < kTable; i += kWalkThreads) {
    const Pair e = pair_of(exp2((double)i * (1.0 / kTable)));
    sh.table[i] = make_float2(e.h, e.l);
  }
  const int live = a.counts ? a.counts[b] : rows;
  const bool counted = live >= 1 && live <= rows;
  const int n = counted ? live : 0;
  if (tid == 0) sh.status = counted ? TV_OK : TV_ERR_INPUT;
  if (tid == 0) sh.removed = 0;
  __syncthreads();
  // 1. the tree: every parent is an earlier node, every drafted token a word
  for (int i = tid; i < n; i += kWalkThreads) {
    int p = 0;
    int64_t t = draft[i];
    if (i > 0) {
      int64_t pr = parent[i - 1];
      if (pr == i - 1) pr = -1;
      if (pr < -1 || pr + 1 >= i || t < 0 || t >= vocab) {
        sh.status = TV_ERR_INPUT;
        t = 0;
      } else {
        p = (int)pr + 1;
      }
    }
    par[i] = p;
    tok[i] = t;
    take[i] = -1;
  }
  __syncthreads();
  const bool bad = sh.status != TV_OK;
  // the drafted words' logits and the draw's number, on their way while stage 1
  // ends; like the tree above they come before this kernel's grid_wait, behind stage 1's
  const float u0 = n > 0 ? u[0] : 0.f;
  float child_logit[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = tid + q * kWalkThreads;
    child_logit[q] = i > 0 && i < n ? as_float<E>(logits[(int64_t)par[i] * a.l_sm + tok[i]]) : 0.f;
  }
  // 2. each node's maximum and normaliser from its chunks' pairs, five nodes'
  // loads at a time (a tree of 64 and its root in one turn)
  constexpr int kNodes = 5;
  grid_wait();
  for (int i0 = warp; i0 < n; i0 += kNodes * kWalkWarps) {
    float m[kNodes], pm[kNodes];
    double ps[kNodes], s[kNodes];
#pragma unroll
    for (int q = 0; q < kNodes; ++q) {
      const int i = i0 + q * kWalkWarps;
      const int64_t at = ((int64_t)b * rows + i) * a.chunks + lane;
      const bool in = i < n && lane < a.chunks;
      pm[q] = in ? a.part_max[at] : -INFINITY;
      ps[q] = in ? a.part_sum[at] : 0.0;
      m[q] = pm[q];
      for (int c = 32; i < n && c + lane < a.chunks; c += 32) m[q] = fmaxf(m[q], a.part_max[at + c]);
    }
#pragma unroll
    for (int q = 0; q < kNodes; ++q) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m[q] = fmaxf(m[q], __shfl_xor_sync(0xffffffffu, m[q], o));
      m[q] = m[q] == -INFINITY ? 0.f : m[q];
      s[q] = ps[q] * (double)weight32(pm[q], m[q], a.c_hi, a.c_lo);
      const int i = i0 + q * kWalkWarps;
      const int64_t at = ((int64_t)b * rows + i) * a.chunks + lane;
      for (int c = 32; i < n && c + lane < a.chunks; c += 32)
        s[q] += a.part_sum[at + c] * (double)weight32(a.part_max[at + c], m[q], a.c_hi, a.c_lo);
    }
#pragma unroll
    for (int q = 0; q < kNodes; ++q) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
      const int i = i0 + q * kWalkWarps;
      if (lane == 0 && i < n) {
        mx[i] = m[q];
        z[i] = s[q];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = tid + q * kWalkThreads;
    if (i < 1 || i >= n) continue;
    const int p = par[i];
    prob[i] = value(weight_pair<true>(child_logit[q], mx[p], a.exponent, sh.table)) / z[p];
    int same = 0;
#pragma unroll 8
    for (int j = p + 1; j < i; ++j) same |= (par[j] == p) & (tok[j] == tok[i]);
    dup[i] = same;
  }
  cluster.sync();     // every CTA of the cluster runs before another writes to its shared memory

  const int first_block = rank * a.blocks;
  const int all_blocks = (vocab + kBlock - 1) / kBlock;
  const int my_blocks = max(0, min(a.blocks, all_blocks - first_block));
  int node = 0, length = 1;
  double qa = 0.0, qb = 1.0;                   // sampled drafts: (p - qa q)+ and its sum
  bool whole = false;                          // draw from p itself
  double left = 0.0;                           // sum of the weights that are drawn from

  Pair za = {0.f, 0.f}, aa = {0.f, 0.f};        // 1 / the row's sum of weights, and qa

  // Logits (and draft probabilities) of words j0 + k * step of a block at the
  // current node: none behind a branch of its own, so that all are in flight
  // together.  Past the end of the vocabulary they are the last word's.
  constexpr bool kExact = sizeof(E) == 4;
  struct Words {
    E l[kLane];
    Q q[kLane];
  };
  auto load_words = [&](int j0, int step, Words& x) {
    const E* row = logits + (int64_t)node * a.l_sm;
    const Q* qrow = static_cast<const Q*>(a.probs) + (int64_t)b * a.q_sb + (int64_t)node * a.q_sm;
    if (j0 + kBlock <= vocab) {
#pragma unroll
      for (int k = 0; k < kLane; ++k) x.l[k] = row[j0 + step * k];
      if (SAMPLED && qa > 0.0 && !whole) {
#pragma unroll
        for (int k = 0; k < kLane; ++k) x.q[k] = qrow[j0 + step * k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < kLane; ++k) x.l[k] = row[min(j0 + step * k, vocab - 1)];
      if (SAMPLED && qa > 0.0 && !whole) {
#pragma unroll
        for (int k = 0; k < kLane; ++k) x.q[k] = qrow[min(j0 + step * k, vocab - 1)];
      }
    }
  };
  // What is left of their weights.
  auto weigh = [&](int j0, int step, const Words& x, Pair* w) {
    const float base = mx[node];
#pragma unroll
    for (int k = 0; k < kLane; ++k) w[k] = weight_pair<kExact>(as_float<E>(x.l[k]), base, a.exponent, sh.table);
    if (SAMPLED && qa > 0.0 && !whole) {
#pragma unroll
      for (int k = 0; k < kLane; ++k) {
        // p - qa q
        const Pair e = w[k];
        const float q = as_float<Q>(x.q[k]);
        const float p = e.h * za.h;
        const float pl = fmaf(e.h, za.l, fmaf(e.l, za.h, fmaf(e.h, za.h, -p)));
        const float t = aa.h * q;
        const float tl = fmaf(aa.l, q, fmaf(aa.h, q, -t));
        const Pair d = two_sum(p, -t);
        const float dl = d.l + (pl - tl), dh = d.h + dl;
        w[k].h = dh < 0.f ? 0.f : dh;
        w[k].l = dh < 0.f ? 0.f : dl - (dh - d.h);
      }
    }
    if (!SAMPLED && !whole) {
      // words taken out of the distribution: few, so first whether this block has any
      const int lo = j0 - lane * (step == 1 ? kLane : 1);
      bool any = false;
      for (int i = lane; i < sh.removed; i += 32) any |= (unsigned)(dup[i] - lo) < (unsigned)kBlock;
      if (__any_sync(0xffffffffu, any)) {
        for (int i = 0; i < sh.removed; ++i)
#pragma unroll
          for (int k = 0; k < kLane; ++k)
            if (dup[i] == j0 + step * k && w[k].l == w[k].l) w[k] = {0.f, 0.f};
      }
    }
    if (j0 + kBlock > vocab) {
#pragma unroll
      for (int k = 0; k < kLane; ++k)
        if (j0 + step * k >= vocab) w[k] = {0.f, 0.f};
    }
  };
  // The eight words' sum, as a pair.
  auto lane_sum = [&](const Pair* w) {
    Pair s = w[0];
#pragma unroll
    for (int k = 1; k < kLane; ++k) {
      const Pair t = two_sum(s.h, w[k].h);
      s = {t.h, s.l + (t.l + w[k].l)};
    }
    const float h = s.h + s.l;
    return Pair{h, s.l - (h - s.h)};
  };
  // Sum over the row: the blocks' sums stay in block_sum, the CTAs' in
  // sh.cta_sum[turn] of every CTA.  The two buffers alternate, so one cluster
  // barrier a round is enough.  A warp's next block is on its way while it
  // sums the present one.
  int turn = 0;
  auto sum_row = [&] {
    __syncthreads();
    Words next;
    load_words((first_block + warp) * kBlock + lane, 32, next);
    for (int t = warp; t < my_blocks; t += kWalkWarps) {
      const Words now = next;
      load_words((first_block + t + kWalkWarps) * kBlock + lane, 32, next);
      Pair w[kLane];
      weigh((first_block + t) * kBlock + lane, 32, now, w);
      const Pair s = warp_sum(lane_sum(w));
      if (lane == 0) block_sum[t] = value(s);
    }
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      double s = 0.0;
      for (int t = lane; t < my_blocks; t += 32) s += block_sum[t];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane < size) *cluster.map_shared_rank(&sh.cta_sum[turn][rank], lane) = s;
    }
    cluster.sync();
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) s += r < size ? sh.cta_sum[turn][r] : 0.0;
    return s;
  };

  if (!bad) {
    if constexpr (!SAMPLED) {
      // 3a. fixed drafts: every child is decided on its own
      for (int i = tid; i < n; i += kWalkThreads) {
        if (i == 0 || dup[i]) continue;
        const int p = par[i];
        double gone = 0.0;
#pragma unroll 8
        for (int j = p + 1; j < i; ++j) gone += par[j] == p && !dup[j] ? prob[j] : 0.0;
        if ((double)u[i] * (1.0 - gone) < prob[i]) atomicMin(reinterpret_cast<unsigned*>(&take[p]), (unsigned)i);
      }
      __syncthreads();
      while (take[node] > 0) {
        node = take[node];
        ++length;
      }
      __syncthreads();              // dup is a list of words from here on
      for (int i = node + 1 + tid; i < n; i += kWalkThreads)
        if (par[i] == node) dup[atomicAdd(&sh.removed, 1)] = (int)tok[i];
    }
    // 3b. sampled drafts: node by node, each rejection a pass over the row (the
    // first one two: the row's own sum, then what is left).  4. The draw's
    // pass, twice where nothing is left: then from the node's own
    // distribution.  One loop, so that the pass's code is there once: run
    // once or twice a launch, it costs as much to fetch as to execute.
    enum { kScan, kRowSum, kRest, kDraw };
    int want = SAMPLED ? kScan : kDraw, i = 1;
    bool summed = false;
    for (;;) {
      if (SAMPLED && want == kScan) {
        for (; i < n; ++i) {
          if (par[i] != node) continue;
          const Q* qrow = static_cast<const Q*>(a.probs) + (int64_t)b * a.q_sb + (int64_t)node * a.q_sm;
          const double q = (double)as_float<Q>(qrow[tok[i]]);
          const double d = prob[i] - (qa > 0.0 ? qa * q : 0.0);
          if (!((double)u[i] * qb * q < (d > 0.0 ? d : 0.0))) break;
          if (tid == 0) take[node] = i;
          node = i;
          ++length;
          qa = 0.0;
          qb = 1.0;
          summed = false;
        }
        if (i == n && summed && left != 0.0) break;
        want = i == n ? kDraw : qa == 0.0 ? kRowSum : kRest;
        if (want == kDraw) whole = summed;
        if (want == kRest) {
          qa += qb;
          aa = pair_of(qa);
        }
      }
      left = sum_row();
      if (SAMPLED && want == kRowSum) {
        za = pair_of(1.0 / left);
        qa = qb;
        aa = pair_of(qa);
        want = kRest;
      } else if (SAMPLED && want == kRest) {
        qb = left;
        summed = true;
        want = kScan;
        ++i;
      } else if (left == 0.0 && !whole) {
        whole = true;
      } else {
        break;
      }
    }
  }
  const bool fail = bad || !(left > 0.0) || left == (double)INFINITY;
  if (!fail) {
    float uf = u0;
    if (!(uf >= 0.f)) uf = 0.f;
    if (!(uf < 1.f)) uf = 0.99999994f;
    const double v = (double)uf * left;
    // the CTA, then the block, then the word at which the cumulated weight
    // first exceeds v; if rounding leaves none, the last one with any weight
    int owner = 0;
    double start = 0.0;
    {
      double at = 0.0;
      bool hit = false;
      for (int r = 0; r < size && !hit; ++r) {
        const double s = sh.cta_sum[turn][r];
        if (s > 0.0) {
          owner = r;
          start = at;
        }
        hit = at + s > v;
        at += s;
      }
    }
    if (rank == owner && warp == 0) {
      int block = 0;
      double at = start;
      {
        double run = start;
        bool hit = false;
        for (int t0 = 0; t0 < my_blocks && !hit; t0 += 32) {
          const double s = t0 + lane < my_blocks ? block_sum[t0 + lane] : 0.0;
          double c = s;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double t = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += t;
          }
          const unsigned over = __ballot_sync(0xffffffffu, s > 0.0 && run + c > v);
          const unsigned some = __ballot_sync(0xffffffffu, s > 0.0);
          hit = over != 0;
          if (some) {
            const int l = over ? __ffs(over) - 1 : 31 - __clz(some);
            block = t0 + l;
            at = run + __shfl_sync(0xffffffffu, c - s, l);
          }
          run += __shfl_sync(0xffffffffu, c, 31);
        }
      }
      // eight consecutive words a lane: one scan over the lanes, then one lane's eight
      Pair w[kLane];
      Words x;
      const int j0 = (first_block + block) * kBlock + lane * kLane;
      load_words(j0, 1, x);
      weigh(j0, 1, x, w);
      int last = -1;                 // this lane's last word with any weight
#pragma unroll
      for (int k = 0; k < kLane; ++k)
        if (w[k].h > 0.f) last = j0 + k;
      const double mine = value(lane_sum(w));
      double c = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += t;
      }
      const unsigned over = __ballot_sync(0xffffffffu, last >= 0 && at + c > v);
      const unsigned some = __ballot_sync(0xffffffffu, last >= 0);
      const int at_lane = over ? __ffs(over) - 1 : 31 - __clz(some);
      double run = at + (c - mine);
      int pick = last;
      bool hit = false;
#pragma unroll
      for (int k = 0; k < kLane; ++k) {
        run += value(w[k]);
        if (!hit && w[k].h > 0.f && run > v) {
          pick = j0 + k;
          hit = true;
        }
      }
      pick = __shfl_sync(0xffffffffu, pick, at_lane);
      if (lane == 0) {
        result[3] = pick;
        next_tokens[node] = pick;
      }
    }
  }
  // 5. the rest of the result
  if (rank == 0) {
    for (int i = tid; i < rows; i += kWalkThreads)
      if (fail || i != node) next_tokens[i] = -1;
    for (int i = tid + (fail ? 0 : length); i < rows; i += kWalkThreads) result[8 + i] = result[8 + rows + i] = -1;
    if (tid == 0) {
      result[0] = fail ? TV_ERR_INPUT : TV_OK;
      result[1] = fail ? 0 : node;
      result[2] = fail ? 0 : length;
      if (fail) result[3] = -1;
      for (int k = 4; k < 8; ++k) result[k] = 0;
      if (!fail) {
        int i = 0;
        for (int at = 0; at < length; ++at) {
          result[8 + at] = i;
          result[8 + rows + at] = tok[i];
          i = take[i];
        }
      }
    }
  }
}

int chunk_elems(int dtype) { return kChunkBytes / (dtype == TV_F32 ? 4 : 2); }
int chunk_count(int dtype, int vocab) { return (vocab + chunk_elems(dtype) - 1) / chunk_elems(dtype); }

// CTAs per sequence: one per 4096 words, as many as run at once (one per SM; as
// the occupancy query reports it, clusters do not span processor groups).  16,
// beyond the portable 8, takes 2 of 21 us off one tree over 128256 words.
int cluster_size(int vocab, int batch) {
  constexpr int fit[9] = {0, 1 << 30, 74, 45, 33, 26, 22, 15, 15};
  if (batch <= 7 && vocab > 8 * 4096) return 16;
  int c = 8;
  while (c > 1 && (batch > fit[c] || (c - 1) * 4096 >= vocab)) --c;
  return c;
}

// Clusters of more than 8 CTAs are opted into once per kernel and device.
template <typename E, typename Q, bool SAMPLED>
int ensure_wide_cluster() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (dev < 64 && (done.load() >> dev & 1)) return TV_OK;
  e = cudaFuncSetAttribute(walk_kernel<E, Q, SAMPLED>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (dev < 64) done.fetch_or(1ull << dev);
  return TV_OK;
}

template <typename E, typename Q, bool SAMPLED>
int launch_walk(const Args& a, int batch, size_t smem, cudaStream_t st) {
  if (smem > 32 * 1024) {
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(walk_kernel<E, Q, SAMPLED>), (int)smem);
    if (rc != TV_OK) return rc;
  }
  const int size = cluster_size(a.vocab, batch);
  if (size > 8) {
    const int rc = ensure_wide_cluster<E, Q, SAMPLED>();
    if (rc != TV_OK) return rc;
  }
  // stage 2 starts while stage 1 ends and waits for its results on the device
  return launch_early(walk_kernel<E, Q, SAMPLED>, dim3((unsigned)size, (unsigned)batch), kWalkThreads, smem, size, st, a);
}

template <typename E>
int launch(const Args& a, int probs_dtype, int batch, size_t smem, cudaStream_t st) {
  const int rc = launch_early(row_stats_kernel<E>, dim3((unsigned)a.chunks, (unsigned)a.rows, (unsigned)batch),
                              kStatThreads, 0, 0, st, a);
  if (rc != TV_OK) return rc;
  if (!a.probs) return launch_walk<E, float, false>(a, batch, smem, st);
  if (probs_dtype == TV_F32) return launch_walk<E, float, true>(a, batch, smem, st);
  if (probs_dtype == TV_F16) return launch_walk<E, __half, true>(a, batch, smem, st);
  return launch_walk<E, __nv_bfloat16, true>(a, batch, smem, st);
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" {

int tv_residual_accept_workspace_size(const tv_residual_accept_args* a, size_t* bytes) {
  if (!a || !bytes) return TV_ERR_NULL;
  if (a->batch < 0 || a->rows < 1 || a->vocab < 1) return TV_ERR_SHAPE;
  const size_t pairs = (size_t)a->batch * a->rows * chunk_count(a->logits_dtype, a->vocab);
  *bytes = pairs * (sizeof(double) + sizeof(float)) + 16;
  return TV_OK;
}

int tv_residual_accept(const tv_residual_accept_args* a, void* stream) {
  if (!a) return TV_ERR_NULL;
  if (a->batch < 0 || a->rows < 1 || a->vocab < 1) return TV_ERR_SHAPE;
  if (a->rows > 1024 || a->batch > 65535 || a->vocab > (1 << 30)) return TV_ERR_UNSUPPORTED;
  if (a->logits_dtype < TV_BF16 || a->logits_dtype > TV_F32) return TV_ERR_DTYPE;
  if (a->probs && (a->probs_dtype < TV_BF16 || a->probs_dtype > TV_F32)) return TV_ERR_DTYPE;
  if (!(a->temperature >= 1e-20) || !(a->temperature <= 1e20)) return TV_ERR_INPUT;   // log2(e) / T as a float
  if (a->batch == 0) return TV_OK;
  if (!a->logits || !a->draft || !a->uniform || !a->next_tokens || !a->result) return TV_ERR_NULL;
  if (a->rows > 1 && !a->parent) return TV_ERR_NULL;
  size_t need = 0;
  tv_residual_accept_workspace_size(a, &need);
  if (!a->workspace || a->workspace_bytes < need) return TV_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return TV_ERR_ALIGN;
  Args k{};
  k.logits = a->logits;
  k.l_sb = a->logits_sb;
  k.l_sm = a->logits_sm;
  k.rows = a->rows;
  k.vocab = a->vocab;
  k.chunk = chunk_elems(a->logits_dtype);
  k.chunks = chunk_count(a->logits_dtype, a->vocab);
  k.draft = a->draft;
  k.d_sb = a->draft_sb;
  k.parent = a->parent;
  k.p_sb = a->parent_sb;
  k.counts = a->counts;
  k.uniform = a->uniform;
  k.u_sb = a->uniform_sb;
  k.probs = a->probs;
  k.q_sb = a->probs_sb;
  k.q_sm = a->probs_sm;
  const double c = 1.4426950408889634074 / a->temperature;
  k.c_hi = (float)c;
  while ((double)k.c_hi >= c) k.c_hi = nextafterf(k.c_hi, 0.f);
  k.c_lo = (float)(c - (double)k.c_hi);
  k.exponent.c.h = (float)(1024.0 * c);
  k.exponent.c.l = (float)(1024.0 * c - (double)k.exponent.c.h);
  k.exponent.floor = (float)(-200.0 / c);
  k.part_sum = static_cast<double*>(a->workspace);
  k.part_max = reinterpret_cast<float*>(k.part_sum + (size_t)a->batch * a->rows * k.chunks);
  k.next_tokens = a->next_tokens;
  k.result = a->result;
  const int words = cluster_size(a->vocab, a->batch) * kBlock;
  k.blocks = (a->vocab + words - 1) / words;
  const size_t smem = (size_t)a->rows * (2 * sizeof(double) + sizeof(int64_t) + sizeof(float) + 3 * sizeof(int)) +
                      (size_t)k.blocks * sizeof(double);
  if (smem > 200 * 1024) return TV_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->logits_dtype) {
    case TV_BF16: return launch<__nv_bfloat16>(k, a->probs_dtype, a->batch, smem, st);
    case TV_F16: return launch<__half>(k, a->probs_dtype, a->batch, smem, st);
    default: return launch<float>(k, a->probs_dtype, a->batch, smem, st);
  }
}

}  // extern "C"
