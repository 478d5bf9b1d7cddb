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
// shared memory.  Whole numbers hang on comparisons here, so stage 2 computes
// weights and sums in 64 bits; stage 1's normaliser (fp32 exponentials summed
// in 64 bits) only enters the comparisons of a child's probability.
#include <cooperative_groups.h>

#include "common.cuh"

namespace tv {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256;
constexpr int kChunkBytes = 16384;      // logits per stage-1 CTA: four 16-byte loads a thread
constexpr int kWalkThreads = 512;
constexpr int kWalkWarps = kWalkThreads / 32;
constexpr int kMaxCluster = 8;

template <typename E> __device__ __forceinline__ float as_float(E x);
template <> __device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float as_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float as_float<float>(float x) { return x; }

// Draft probabilities come in any of the three types, chosen at run time.
__device__ __forceinline__ double load_prob(const void* p, int dtype, int64_t i) {
  if (dtype == TV_F32) return (double)static_cast<const float*>(p)[i];
  if (dtype == TV_F16) return (double)__half2float(static_cast<const __half*>(p)[i]);
  return (double)__bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
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
  int probs_dtype;
  int64_t q_sb, q_sm;
  double inv_t;
  float c_hi, c_lo;            // log2(e) / T as a sum of two floats
  float* part_max;             // [batch][rows][chunks]
  double* part_sum;
  int64_t* next_tokens;        // [batch][rows]
  int64_t* result;             // [batch][8 + 2 rows]
};

// exp((l - m) / T) in fp32: the product with log2(e) / T carries its rounding
// error along, so the result is within a few 2^-23 at any magnitude.
__device__ __forceinline__ float weight32(float l, float m, float c_hi, float c_lo) {
  const float x = l - m;
  const float t = x * c_hi;
  const float r = fmaf(x, c_lo, fmaf(x, c_hi, -t));
  const float e = fast_exp2(t);
  return x == -INFINITY ? 0.f : fmaf(e, r * kLn2, e);
}

template <typename E>
__global__ void __launch_bounds__(kStatThreads) row_stats_kernel(const Args a) {
  constexpr int VEC = 16 / sizeof(E);
  constexpr int U = kChunkBytes / (16 * kStatThreads);
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
constexpr int kMarks = 64;              // 2048 marks of removed words, by word mod 2048

struct Walk {
  double cta_sum[2][kMaxCluster];
  uint32_t mark[kMarks];
  int status;
};

template <typename E>
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
  const int live = a.counts ? a.counts[b] : rows;
  const bool counted = live >= 1 && live <= rows;
  const int n = counted ? live : 0;
  if (tid == 0) sh.status = counted ? TV_OK : TV_ERR_INPUT;
  if (tid < kMarks) sh.mark[tid] = 0;
  __syncthreads();
  // 1. the tree: every parent is an earlier node, every drafted token a word
  for (int i = tid; i < n; i += kWalkThreads) {
    int p = 0;
    int64_t t = draft[i];
    if (i > 0) {
      const int64_t pr = parent[i - 1];
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
  // 2. each node's maximum and normaliser from its chunks' pairs
  for (int i = warp; i < n; i += kWalkWarps) {
    const int64_t at = ((int64_t)b * rows + i) * a.chunks;
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, a.part_max[at + c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    double s = 0.0;
    for (int c = lane; c < a.chunks; c += 32)
      s += a.part_sum[at + c] * exp(((double)a.part_max[at + c] - (double)base) * a.inv_t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      mx[i] = base;
      z[i] = s;
    }
  }
  __syncthreads();
  const bool bad = sh.status != TV_OK;
  for (int i = tid; i < n; i += kWalkThreads) {
    if (i == 0) continue;
    const int p = par[i];
    const double l = (double)as_float<E>(logits[(int64_t)p * a.l_sm + tok[i]]);
    prob[i] = exp((l - (double)mx[p]) * a.inv_t) / z[p];
    int same = 0;
    for (int j = p + 1; j < i; ++j) same |= par[j] == p && tok[j] == tok[i];
    dup[i] = same;
  }
  cluster.sync();     // every CTA of the cluster runs before another writes to its shared memory

  const int first_block = rank * a.blocks;
  const int all_blocks = (vocab + kBlock - 1) / kBlock;
  const int my_blocks = max(0, min(a.blocks, all_blocks - first_block));
  int node = 0, length = 1;
  double qa = 0.0, qb = 1.0, zq = 0.0;       // sampled drafts: (p - qa q)+, its sum; the row's exact normaliser
  bool whole = false;                          // draw from p itself
  double left = 0.0;                           // sum of the weights that are drawn from
  bool summed = false;

  // What is left at the current node of the weights of words j0 + 32 k + lane.
  auto weights = [&](int j0, double* w) {
    const E* row = logits + (int64_t)node * a.l_sm;
    const int64_t qoff = (int64_t)b * a.q_sb + (int64_t)node * a.q_sm;
    const double base = (double)mx[node];
    const bool minus = a.probs && qa > 0.0 && !whole;
    float l[kLane];
    double q[kLane];
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      const int j = j0 + 32 * k + lane;
      l[k] = j < vocab ? as_float<E>(row[j]) : -INFINITY;
      q[k] = minus && j < vocab ? load_prob(a.probs, a.probs_dtype, qoff + j) : 0.0;
    }
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      const int j = j0 + 32 * k + lane;
      double e = exp(((double)l[k] - base) * a.inv_t);
      if (minus) {
        const double d = e / zq - qa * q[k];
        e = d < 0.0 ? 0.0 : d;
      } else if (!a.probs && !whole && j < vocab && ((sh.mark[(j >> 5) & (kMarks - 1)] >> (j & 31)) & 1)) {
        for (int i = node + 1; i < n; ++i)
          if (par[i] == node && tok[i] == j && e == e) e = 0.0;
      }
      w[k] = e;
    }
  };
  // Sum over the row: the blocks' sums stay in block_sum, the CTAs' in
  // sh.cta_sum[turn] of every CTA.  The two buffers alternate, so one cluster
  // barrier a round is enough.
  int turn = 0;
  auto sum_row = [&] {
    __syncthreads();
    for (int t = warp; t < my_blocks; t += kWalkWarps) {
      double w[kLane], s = 0.0;
      weights((first_block + t) * kBlock, w);
#pragma unroll
      for (int k = 0; k < kLane; ++k) s += w[k];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) block_sum[t] = s;
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
    for (int r = 0; r < size; ++r) s += sh.cta_sum[turn][r];
    return s;
  };

  if (!bad) {
    if (!a.probs) {
      // 3a. fixed drafts: every child is decided on its own
      for (int i = tid; i < n; i += kWalkThreads) {
        if (i == 0 || dup[i]) continue;
        const int p = par[i];
        double gone = 0.0;
        for (int j = p + 1; j < i; ++j)
          if (par[j] == p && !dup[j]) gone += prob[j];
        if ((double)u[i] * (1.0 - gone) < prob[i]) atomicMin(reinterpret_cast<unsigned*>(&take[p]), (unsigned)i);
      }
      __syncthreads();
      while (take[node] > 0) {
        node = take[node];
        ++length;
      }
      for (int i = node + 1 + tid; i < n; i += kWalkThreads)
        if (par[i] == node) atomicOr(&sh.mark[(tok[i] >> 5) & (kMarks - 1)], 1u << (tok[i] & 31));
    } else {
      // 3b. sampled drafts: node by node, each rejection a pass over the row
      for (int i = 1; i < n; ++i) {
        if (par[i] != node) continue;
        const double q = load_prob(a.probs, a.probs_dtype, (int64_t)b * a.q_sb + (int64_t)node * a.q_sm + tok[i]);
        const double d = prob[i] - (qa > 0.0 ? qa * q : 0.0);
        if ((double)u[i] * qb * q < (d > 0.0 ? d : 0.0)) {
          if (tid == 0) take[node] = i;
          node = i;
          ++length;
          qa = 0.0;
          qb = 1.0;
          summed = false;
        } else {
          if (qa == 0.0) zq = sum_row();
          qa += qb;
          left = qb = sum_row();
          summed = true;
        }
      }
    }
    // 4. the draw: from the node's own distribution where nothing is left
    if (!summed) left = sum_row();
    if (left == 0.0) {
      whole = true;
      left = sum_row();
    }
  }
  const bool fail = bad || !(left > 0.0) || left == (double)INFINITY;
  if (!fail) {
    float uf = u[0];
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
      double w[kLane];
      const int j0 = (first_block + block) * kBlock;
      weights(j0, w);
      int pick = j0;
      bool hit = false;
#pragma unroll
      for (int k = 0; k < kLane; ++k) {
        double c = w[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double t = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) c += t;
        }
        const unsigned over = __ballot_sync(0xffffffffu, w[k] > 0.0 && at + c > v);
        const unsigned some = __ballot_sync(0xffffffffu, w[k] > 0.0);
        if (!hit && some) pick = j0 + 32 * k + (over ? __ffs(over) - 1 : 31 - __clz(some));
        hit |= over != 0;
        at += __shfl_sync(0xffffffffu, c, 31);
      }
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

// CTAs per sequence: one per 4096 words, up to the portable cluster size.
int cluster_size(int vocab) {
  int c = 1;
  while (c < kMaxCluster && c * 4096 < vocab) c *= 2;
  return c;
}

template <typename E>
int launch(const Args& a, int batch, size_t smem, cudaStream_t st) {
  row_stats_kernel<E><<<dim3(a.chunks, a.rows, batch), kStatThreads, 0, st>>>(a);
  int rc = check_launch();
  if (rc != TV_OK) return rc;
  if (smem > 40 * 1024) {
    rc = ensure_dynamic_smem(reinterpret_cast<const void*>(walk_kernel<E>), (int)smem);
    if (rc != TV_OK) return rc;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(cluster_size(a.vocab), batch);
  cfg.blockDim = dim3(kWalkThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster_size(a.vocab);
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, walk_kernel<E>, a);
  return e == cudaSuccess ? check_launch() : record_cuda_error(e);
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
  if (!(a->temperature > 0.f) || !(a->temperature <= 3.4e38f)) return TV_ERR_INPUT;
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
  k.probs_dtype = a->probs_dtype;
  k.q_sb = a->probs_sb;
  k.q_sm = a->probs_sm;
  k.inv_t = 1.0 / (double)a->temperature;
  const double c = 1.4426950408889634074 / (double)a->temperature;
  k.c_hi = (float)c;
  k.c_lo = (float)(c - (double)k.c_hi);
  k.part_sum = static_cast<double*>(a->workspace);
  k.part_max = reinterpret_cast<float*>(k.part_sum + (size_t)a->batch * a->rows * k.chunks);
  k.next_tokens = a->next_tokens;
  k.result = a->result;
  const int words = cluster_size(a->vocab) * kBlock;
  k.blocks = (a->vocab + words - 1) / words;
  const size_t smem = (size_t)a->rows * (2 * sizeof(double) + sizeof(int64_t) + sizeof(float) + 3 * sizeof(int)) +
                      (size_t)k.blocks * sizeof(double);
  if (smem > 200 * 1024) return TV_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->logits_dtype) {
    case TV_BF16: return launch<__nv_bfloat16>(k, a->batch, smem, st);
    case TV_F16: return launch<__half>(k, a->batch, smem, st);
    default: return launch<float>(k, a->batch, smem, st);
  }
}

}  // extern "C"
