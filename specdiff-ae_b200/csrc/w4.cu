// Rows times 4-bit weights with group scales (sm_100a):
//
//   y[t, n] = xs[t] * sum_k x[t, k] * (u[n, k] - 8) * s[n, k / group]
//
// A CTA takes 128 weight rows (the M of tcgen05.mma, one TMEM lane each), up
// to 128 tokens (its N) and a range of k.  The packed weights stream through a
// shared-memory ring (TMA, 128 rows x 256 k = 16 KB a stage).  Eight warps, two
// groups of four, turn them into 16-bit values, a thread one half of a stage
// of its own weight row, and write those straight into tensor memory, where
// the MMA reads its A operand; x comes by TMA as the B operand in tiles of
// 128 k.
//
//   warp 0      weight producer (TMA)
//   warp 1      MMA issuer, tensor-memory owner
//   warp 2      x producer (TMA)
//   warps 4-11  weights to 16 bits (group w / 4 - 1 takes that half of every
//               stage), then the epilogue (TMEM lane quarter w mod 4)
//
// Where there are fewer tiles than CTAs that fit the GPU, a cluster of up to 8
// CTAs splits k; the partial sums meet in distributed shared memory and are
// added in rank order, so results do not depend on timing.
//
// Each (u - 8) * s is rounded once to x's 16-bit type (the MMA takes no other):
// half a step, as the weight itself had in that type.  The error against 64
// bits is 0.0022 in bf16 and 0.00028 in fp16 with it, 0.0017 and 0.00021 for an
// unrounded weight (the output's own rounding).
//
// What bounds it: an MMA of 128 rows x 16 k takes about 37 cycles however few
// the tokens (its A operand's way out of tensor memory), so a stage is 0.32 us of
// an SM's tensor pipe, and two CTAs there were seen to take 0.37 a stage: 65
// rows x 28672 x 4096 (21.8 us) spend 12 us in that (16 stages, two CTAs on half
// of the SMs, one on the others), the rest on the way to the first weights (2-3)
// and from the last MMA to the stored rows (2).  128 rows x 128256 x 4096: 119 us,
// 1.13 PFLOP/s, and 136 once the power cap has the SMs at 1.6 GHz.  Where k is split, 65 rows x 4096 x 14336 take 16.0 us, 4 of them
// behind the last MMA: two cluster barriers and the sums' way between SMs.
// Tiles of 256 weight rows with k cut evenly over the SMs balance better and were
// slower, as were pairs of CTAs splitting k (37 us at 28672 x 4096): partial sums
// cost more than idle SMs.  Weights as the B operand would pad the tokens to 128.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_fp8.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "sm100.cuh"
#include "w4.cuh"

namespace tv {
namespace {

using namespace sm100;
using namespace w4;
namespace cg = cooperative_groups;

constexpr int kRows = 128;                   // weight rows per CTA
constexpr int kMaxTokens = 128;              // tokens per CTA
constexpr int kHalfK = 128;                  // k per x tile, A buffer and group step
constexpr int kStageK = 2 * kHalfK;          // k per weight stage
constexpr int kWStage = kRows * kStageK / 2; // 16 KB
constexpr int kThreads = 384;
constexpr int kDequantWarp = 4;              // first of the eight
constexpr int kMaxStages = 8;
constexpr int kRing = 112 * 1024;            // both rings: two CTAs share an SM
constexpr int kSmem = kRing + 1024;
constexpr uint32_t kTmemCols = 256;          // two CTAs per SM
constexpr uint32_t kACol = 128;              // accumulator in columns 0-127, two 64-column A buffers after it
constexpr int kMaxCluster = 8;

struct Bars {
  uint64_t w_full[kMaxStages], w_empty[kMaxStages];
  uint64_t x_full[kMaxStages], x_empty[kMaxStages];
  uint64_t a_full[2], a_empty[2];
  uint64_t done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Bars) <= kSmem - kRing, "barrier block");

struct W4Params {
  const void* s;
  int64_t s_sn;
  const float* x_scale;
  void* out;
  int64_t o_sm;
  int rows, n, k, groups;
  int tokens;                  // N of the MMA: tokens per CTA, a multiple of 16
  int w_stages, x_stages, x_bytes;
  int split;                   // CTAs of a cluster
  int* status;                 // optional
  uint32_t zero;               // 0, unknown to the compiler
  uint32_t group_magic;        // k / group = (k / 32) * magic >> 32; 0: group 32
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}

// What ran out, in *status: a producer's wait for a free stage, the MMA
// issuer's for its operands, the unpacking's for weights or a free buffer, the
// epilogue's for the accumulator.
enum { kGaveUpLoads = 1, kGaveUpMma, kGaveUpUnpack, kGaveUpSums };

// The address of a shared-memory word in another CTA of the cluster, and a load
// from there; 0 where `in` is false.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, bool in) {
  float v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t@p ld.shared::cluster.f32 %0, [%1];\n\t}"
               : "=f"(v) : "r"(addr), "r"((uint32_t)in) : "memory");
  return v;
}

// Loads in flight land before shared memory is reused or released: a producer
// ends by waiting for its last loads whatever the abort flag says, 0.2 s each.
__device__ __forceinline__ void drain(uint64_t* full, int stages, int it) {
  volatile int keep_waiting = 0;
  for (int j = it > stages ? it - stages : 0; j < it; ++j)
    mbar_wait_suspend(&full[j % stages], (j / stages) & 1, &keep_waiting, 400000000ll);
}

// A thread reads the scales of its own row, so a warp's load touches 32 rows:
// 32 sectors however little of each it takes.  SCALES says how few loads do:
//   0  group a multiple of 128, rows on the 16-byte grid: one scale a half
//      stage, eight fetched at a time (one load in four stages at group 128)
//   1, 2  group 32 or 64, rows on the 8- or 4-byte grid: one load a half stage
//   3  anything else: each 32 k on its own
template <typename T, int SCALES>
__global__ void __launch_bounds__(kThreads, 2)
    w4_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx, const W4Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars* bars = reinterpret_cast<Bars*>(smem + kRing);
  volatile int* abort = &bars->abort;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  grid_next();
  const int rank = blockIdx.x % p.split;
  const int n0 = blockIdx.x / p.split * kRows;
  const int t0 = blockIdx.y * p.tokens;
  // this CTA's weight stages
  const int all = (p.k + kStageK - 1) / kStageK;
  const int kb0 = (int)((int64_t)all * rank / p.split);
  const int nb = (int)((int64_t)all * (rank + 1) / p.split) - kb0;
  uint8_t* w_ring = smem;
  uint8_t* x_ring = smem + p.w_stages * kWStage;

  // ---- producers' state.  A thread keeps about one TMA box in flight, so a
  // warp's lanes take turns issuing.
  const bool wt = warp == 0;
  uint64_t* full = wt ? bars->w_full : bars->x_full;
  uint64_t* empty = wt ? bars->w_empty : bars->x_empty;
  const int ring = wt ? p.w_stages : p.x_stages, count = wt ? nb : 2 * nb;
  int pi = 0, ps = 0, pph = 1;
  auto issue = [&] {
    if (lane == (pi & 31)) {
      if (wt) {
        mbar_arrive_expect_tx(&full[ps], kWStage);
        tma_load_2d(w_ring + ps * kWStage, &tmw, &full[ps], (kb0 + pi) * (kStageK / 2), n0);
      } else {
        mbar_arrive_expect_tx(&full[ps], p.x_bytes);
        tma_load_3d(x_ring + ps * p.x_bytes, &tmx, &full[ps], 0, t0, 4 * kb0 + 2 * pi);
      }
    }
    __syncwarp();
    if (++ps == ring) {
      ps = 0;
      pph ^= 1;
    }
    ++pi;
  };
  if (wt || warp == 2) {
    // each producer sets up its own barriers and fills its ring before the
    // CTA meets: the first loads run while tensor memory is allocated
    if (lane == 0) {
      prefetch_tmap(wt ? &tmw : &tmx);
      for (int i = 0; i < ring; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], wt ? 8 : 1);
      }
      mbar_fence_init();
    }
    __syncwarp();
    // the first weights may come to L2 before the predecessor's end: what it
    // still writes is seen there all the same
    if (wt && lane < min(count, ring)) tma_prefetch_2d(&tmw, (kb0 + lane) * (kStageK / 2), n0);
    grid_wait();
    while (pi < count && pi < ring) issue();
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars->a_full[i], 4);
        mbar_init(&bars->a_empty[i], 1);
      }
      mbar_init(&bars->done, 1);
      bars->abort = 0;
      mbar_fence_init();
    }
    __syncwarp();
    // not before: a predecessor may still want tensor memory itself, and would
    // wait for what this CTA held while it waits for the predecessor
    grid_wait();
    tmem_alloc(&bars->tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  grid_wait();

  if (wt || warp == 2) {
    while (pi < count) {
      if (!__all_sync(0xffffffffu, mbar_wait_suspend(&empty[ps], pph, abort))) {
        give_up(abort, p.status, kGaveUpLoads);
        break;
      }
      issue();
    }
    if (lane == 0) drain(full, ring, pi);
  } else if (warp == 1) {
    // ---- MMA issuer: the whole warp walks the loop, one elected lane issues
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc = idesc_f16(fmt, kRows, (uint32_t)p.tokens, 0);
    const uint64_t desc0 = smem_desc_sw128(smem_u32(x_ring), 16, 1024);
    const uint32_t half_tile = (uint32_t)p.x_bytes >> 5;          // 64 k of x, in descriptor units
    const bool elected = elect_one();
    int xs = 0, xph = 0;
    bool ok = true;
    for (int i = 0; i < 2 * nb; ++i) {
      const int g = i & 1;
      if (!mbar_wait_suspend(&bars->x_full[xs], xph, abort) ||
          !mbar_wait_suspend(&bars->a_full[g], (i >> 1) & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t b = desc0 + (uint32_t)((xs * p.x_bytes) >> 4);
      const uint32_t a = tmem + kACol + (uint32_t)(g * 64);
      if (elected) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts(tmem, a + kk * 8, b + (kk >> 2) * half_tile + (kk & 3) * 2, idesc, (i | kk) ? 1u : 0u);
        tc_commit(&bars->a_empty[g]);
        tc_commit(&bars->x_empty[xs]);
      }
      __syncwarp();
      if (++xs == p.x_stages) {
        xs = 0;
        xph ^= 1;
      }
    }
    if (!ok) give_up(abort, p.status, kGaveUpMma);
    else if (elected) tc_commit(&bars->done);
  } else if (warp >= kDequantWarp) {
    const int g = (warp - kDequantWarp) >> 2;
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;                        // weight row = TMEM lane
    const uint32_t lanes = tmem + ((uint32_t)(q4 * 32) << 16);
    const uint32_t a_buf = lanes + kACol + (uint32_t)(g * 64);
    const T* row = static_cast<const T*>(p.s) + (int64_t)min(n0 + r, p.n - 1) * p.s_sn;
    const int last = p.k / 32 - 1;                       // last 32-k unit
    auto index = [&](int u) { return p.group_magic ? __umulhi((uint32_t)u, p.group_magic) : (uint32_t)u; };
    constexpr int NS = SCALES == 0 ? 1 : SCALES == 2 ? 2 : 4;     // scales of a half row of a stage
    // The bits that hold the scales of stage st, loaded one stage ahead
    // and only taken apart there, so nothing waits for a load in flight.  Past
    // the end of the weight they are those of its last row (not stored) and
    // last group (its x is zero).
    struct Raw {
      uint32_t v[4];
    };
    auto load_scales = [&](int st, Raw& o) {
      if constexpr (SCALES == 0) {
        const T* at = row + (index(min(st * 8 + g * 4, last)) & ~7u);
        // the last eight of a row that does not end on eight
        if (at + 8 <= row + p.groups)
          asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(o.v[0]), "=r"(o.v[1]), "=r"(o.v[2]), "=r"(o.v[3]) : "l"(at));
        else {
          for (int j = 0; j < 4; ++j) {
            const uint16_t lo = 2 * j < row + p.groups - at ? reinterpret_cast<const uint16_t*>(at)[2 * j] : 0;
            const uint16_t hi = 2 * j + 1 < row + p.groups - at ? reinterpret_cast<const uint16_t*>(at)[2 * j + 1] : 0;
            o.v[j] = (uint32_t)hi << 16 | lo;
          }
        }
      } else if constexpr (SCALES == 1) {
        const T* at = row + min(st * 8 + g * 4, (last / 4) * 4);
        asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(o.v[0]), "=r"(o.v[1]) : "l"(at));
      } else if constexpr (SCALES == 2) {
        const T* at = row + min(st * 4 + g * 2, (last / 4) * 2);
        asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(o.v[0]) : "l"(at));
      } else {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const T* at = row + index(min(st * 8 + g * 4 + b, last));
          asm volatile("{\n\t.reg .u16 t;\n\tld.global.nc.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(o.v[b]) : "l"(at));
        }
      }
    };
    // scale b of the half stage, its bits in both halves
    auto scale_of = [&](const Raw& o, int st, int b) -> uint32_t {
      if constexpr (SCALES == 0) {
        const int u = min(st * 8 + g * 4, last);
        const uint32_t i = index(u) & 7;
        const uint32_t w = (i & 4) ? ((i & 2) ? o.v[3] : o.v[2]) : ((i & 2) ? o.v[1] : o.v[0]);
        return __byte_perm(w, w, (i & 1) ? 0x3232 : 0x1010);
      } else if constexpr (SCALES == 1 || SCALES == 2) {
        return __byte_perm(o.v[b >> 1], 0, (b & 1) ? 0x3232 : 0x1010);
      } else {
        return o.v[b] * 0x10001u;
      }
    };
    Raw raw;
    load_scales(kb0, raw);
    int s = 0, ph = 0;
    bool ok = true;
    for (int i = 0; i < nb; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_suspend(&bars->w_full[s], ph, abort))) {
        ok = false;
        break;
      }
      uint4 w[4];
      const uint8_t* src = w_ring + s * kWStage + r * 128;
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const uint4*>(src + (((g * 4 + c) ^ (r & 7)) << 4));
      // Release the stage once the loads have come back: an arrival may pass
      // loads that are still on their way, and the next TMA write with it, so
      // its address is made to depend on a word of each (p.zero is 0).
      const uint32_t seen = (w[0].x ^ w[1].x ^ w[2].x ^ w[3].x) & p.zero;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->w_empty[s] + seen);
      Unpack<T> un[NS];
#pragma unroll
      for (int b = 0; b < NS; ++b) un[b].scale(scale_of(raw, kb0 + i, b));
      // eight scales at once last until their index leaves the eight
      const int u = (kb0 + i + 1) * 8 + g * 4;
      if (SCALES != 0 || ((index(u) ^ index(u - 8)) & ~7u)) load_scales(kb0 + i + 1, raw);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t o[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const Unpack<T>& u = un[NS == 1 ? 0 : NS == 2 ? h : h * 2 + c];
          const uint4 v = w[h * 2 + c];
          u.word(v.x, o + c * 16);
          u.word(v.y, o + c * 16 + 4);
          u.word(v.z, o + c * 16 + 8);
          u.word(v.w, o + c * 16 + 12);
        }
        if (h == 0) {
          // the MMAs that read this buffer's previous contents have finished
          if (i >= 1 && !__all_sync(0xffffffffu, mbar_wait_suspend(&bars->a_empty[g], (i & 1) ^ 1, abort))) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        tmem_st32(a_buf + (uint32_t)(h * 32), o);
      }
      if (!ok) break;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->a_full[g]);
      if (++s == p.w_stages) {
        s = 0;
        ph ^= 1;
      }
    }
    if (!ok) give_up(abort, p.status, kGaveUpUnpack);
    // ---- epilogue
    ok = __all_sync(0xffffffffu, mbar_wait_suspend(&bars->done, 0, abort)) && ok;
    if (!ok) give_up(abort, p.status, kGaveUpSums);
    tc_fence_after();
    T* out = static_cast<T*>(p.out);
    float* part = reinterpret_cast<float*>(smem);        // [token][weight row], once both rings are drained
    const bool in = n0 + r < p.n;
#pragma unroll 1
    for (int c = g; c * 16 < p.tokens; c += 2) {
      uint32_t v[16];
      tmem_ld16(lanes + (uint32_t)(c * 16), v);
      tmem_wait_ld();
      const int t = t0 + c * 16, left = in ? p.rows - t : 0;
      float f[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] = ok ? __uint_as_float(v[j]) * Unpack<T>::unscale() : __int_as_float(0x7fc00000);
      // no branch per token: each costs what a store does
      if (p.split > 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c * 16 + j) * kRows + r] = f[j];
        continue;
      }
      if (p.x_scale) {
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] *= __ldg(p.x_scale + min(t + j, p.rows - 1));
      }
      T* at = out + (int64_t)t * p.o_sm + n0 + r;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j < left) *at = Elem<T>::from_f(f[j]);
        at += p.o_sm;
      }
    }
  }
  __syncwarp();
  if (p.split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    // a CTA that gave up leaves NaNs, written once its last loads have landed
    if (__syncthreads_or(*abort))
      for (int e = threadIdx.x; e < p.tokens * kRows; e += kThreads)
        reinterpret_cast<float*>(smem)[e] = __int_as_float(0x7fc00000);
    cluster.sync();
    if (warp >= kDequantWarp) {
      const int tid = threadIdx.x - kDequantWarp * 32;
      const int r = tid & (kRows - 1);
      T* out = static_cast<T*>(p.out);
      uint32_t part[kMaxCluster];            // this row's sums in every CTA
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) part[k] = map_rank(smem_u32(smem) + r * 4, min(k, p.split - 1));
      // this CTA's tokens, one of every p.split; three at a time, all of their
      // parts on their way together
      const int step = p.split * 2;
#pragma unroll 1
      for (int j0 = rank + p.split * (tid / kRows); j0 < p.tokens; j0 += 3 * step) {
        float v[3][kMaxCluster];
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int k = 0; k < kMaxCluster; ++k)
            v[i][k] = ld_cluster(part[k] + (j0 + i * step) * (kRows * 4), k < p.split && j0 + i * step < p.tokens);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const int j = j0 + i * step, t = t0 + j;
          float f = 0.f;
#pragma unroll
          for (int k = 0; k < kMaxCluster; ++k) f += v[i][k];
          if (p.x_scale) f *= __ldg(p.x_scale + min(t, p.rows - 1));
          if (j < p.tokens && t < p.rows && n0 + r < p.n) out[(int64_t)t * p.o_sm + n0 + r] = Elem<T>::from_f(f);
        }
      }
    }
    cluster.sync();     // no CTA leaves while another still reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// x that TMA cannot read as it is -> dense 16-bit rows of a multiple of 64,
// zeros behind k: 8-bit rows (both 16-bit types hold every e4m3 value exactly),
// rows off the 16-byte grid, and rows that end inside a 64-k tile.
__host__ __device__ constexpr int padded_k(int k) { return (k + 63) / 64 * 64; }

template <typename X, typename T>
__global__ void __launch_bounds__(256) w4_stage_kernel(const X* x, int64_t x_sm, T* y, int rows, int k) {
  grid_next();
  grid_wait();
  const int chunks = padded_k(k) / 8;
  const int64_t total = (int64_t)rows * chunks;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int64_t r = e / chunks;
    const int c = (int)(e - r * chunks) * 8;
    const X* src = x + r * x_sm + c;
    float f[8] = {};
    if (c < k) {
      if (sizeof(X) == 1 && (reinterpret_cast<uintptr_t>(src) & 7) == 0) {
        const uint2 raw = *reinterpret_cast<const uint2*>(src);
        const X* b = reinterpret_cast<const X*>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(src[i]);
      }
    }
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Elem<T>::pack2(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(y + r * padded_k(k) + c) = o;
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

bool make_map(CUtensorMap* map, CUtensorMapDataType dt, int dims, const void* base, const cuuint64_t* size,
              const cuuint64_t* stride_bytes, const cuuint32_t* box) {
  auto enc = encoder();
  const cuuint32_t one[3] = {1, 1, 1};
  return enc && enc(map, dt, dims, const_cast<void*>(base), size, stride_bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether x goes through the staging copy; one row needs no stride of its own.
bool staged(const tv_w4_args* a) {
  return a->x_dtype == TV_E4M3 || a->k % 64 != 0 || !aligned16(a->x) ||
         (a->rows > 1 && (a->x_sm < a->k || a->x_sm % 8 != 0));
}

template <typename T, int SCALES>
int launch_kernel(const CUtensorMap& mw, const CUtensorMap& mx, const W4Params& p, int blocks_n, int blocks_t,
                  cudaStream_t st) {
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(w4_kernel<T, SCALES>), kSmem);
  if (rc != TV_OK) return rc;
  return launch_early(w4_kernel<T, SCALES>, dim3((unsigned)(blocks_n * p.split), (unsigned)blocks_t), kThreads, kSmem,
                      p.split, st, mw, mx, p);
}

template <typename T>
int launch_w4(const tv_w4_args* a, cudaStream_t st) {
  const void* x = a->x;
  int64_t x_sm = a->rows > 1 ? a->x_sm : padded_k(a->k);
  if (staged(a)) {
    T* y = static_cast<T*>(a->workspace);
    const int64_t chunks = (int64_t)a->rows * (padded_k(a->k) / 8);
    const int blocks = (int)(chunks / 256 + 1 < 4 * kNumSMs ? chunks / 256 + 1 : 4 * kNumSMs);
    const int rc =
        a->x_dtype == TV_E4M3
            ? launch_early(w4_stage_kernel<__nv_fp8_e4m3, T>, dim3((unsigned)blocks), 256, 0, 0, st,
                           static_cast<const __nv_fp8_e4m3*>(a->x), a->x_sm, y, a->rows, a->k)
            : launch_early(w4_stage_kernel<T, T>, dim3((unsigned)blocks), 256, 0, 0, st, static_cast<const T*>(a->x),
                           a->x_sm, y, a->rows, a->k);
    if (rc != TV_OK) return rc;
    x = y;
    x_sm = padded_k(a->k);
  }
  W4Params p{};
  p.s = a->scales;
  p.s_sn = a->s_sn;
  p.x_scale = a->x_dtype == TV_E4M3 ? a->x_scale : nullptr;
  p.out = a->out;
  p.o_sm = a->o_sm;
  p.rows = a->rows;
  p.n = a->n;
  p.k = a->k;
  p.groups = a->k / a->group;
  p.tokens = a->rows >= kMaxTokens ? kMaxTokens : (a->rows + 15) / 16 * 16;
  p.x_bytes = p.tokens * kHalfK * 2;
  // rings: x tiles to cover an L2 round trip, the rest to the weights (3 to 5 stages)
  p.x_stages = p.tokens <= 16 ? 6 : p.tokens <= 48 ? 4 : p.tokens <= 80 ? 3 : 2;
  p.w_stages = (kRing - p.x_stages * p.x_bytes) / kWStage;
  p.group_magic = group_magic(a->group);
  p.status = a->status;
  const int blocks_t = (a->rows + p.tokens - 1) / p.tokens;
  const int64_t tiles = (int64_t)((a->n + kRows - 1) / kRows) * blocks_t;
  const int stages = (a->k + kStageK - 1) / kStageK;
  // the largest cluster of which that many run at once, two CTAs per SM: by the
  // time over the number of tiles (8192 k, 33 rows), which steps from 11.4 to 17.1
  // us behind 33 clusters of 8, 12.3 to 18.7 behind 37 of 7, and so on behind 45
  // of 6, 56 of 5, 70 of 4 and 92 of 3 (clusters do not span processor groups).
  // A little less here, as the groups' sizes differ from one GPU to the next.
  constexpr int fit[kMaxCluster + 1] = {0, 296, 148, 90, 68, 54, 44, 36, 32};
  p.split = 1;
  for (int c = 2; c <= kMaxCluster; ++c)
    if (tiles <= fit[c] && stages >= c) p.split = c;
  CUtensorMap mw, mx;
  const cuuint64_t w_size[2] = {(cuuint64_t)a->k / 2, (cuuint64_t)a->n}, w_stride[1] = {(cuuint64_t)a->q_sn * 4};
  const cuuint32_t w_box[2] = {kStageK / 2, kRows};
  // x as [k / 64][rows][64]: one box is a 128-k tile, each 64 k of it 128-byte swizzled rows
  const cuuint64_t x_size[3] = {64, (cuuint64_t)a->rows, (cuuint64_t)padded_k(a->k) / 64};
  const cuuint64_t x_stride[2] = {(cuuint64_t)x_sm * 2, 128};
  const cuuint32_t x_box[3] = {64, (cuuint32_t)p.tokens, kHalfK / 64};
  const CUtensorMapDataType dt = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (!make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a->qweight, w_size, w_stride, w_box) ||
      !make_map(&mx, dt, 3, x, x_size, x_stride, x_box))
    return TV_ERR_UNSUPPORTED;
  const int blocks_n = (a->n + kRows - 1) / kRows;
  // SCALES by what the layout allows; k a multiple of 128 keeps a half stage's
  // load inside the row
  auto grid_of = [&](int bytes) {
    return reinterpret_cast<uintptr_t>(a->scales) % bytes == 0 && (a->n == 1 || a->s_sn * 2 % bytes == 0);
  };
  if (a->group % kHalfK == 0 && grid_of(16)) return launch_kernel<T, 0>(mw, mx, p, blocks_n, blocks_t, st);
  if (a->group == 32 && a->k % kHalfK == 0 && grid_of(8)) return launch_kernel<T, 1>(mw, mx, p, blocks_n, blocks_t, st);
  if (a->group == 64 && a->k % kHalfK == 0 && grid_of(4)) return launch_kernel<T, 2>(mw, mx, p, blocks_n, blocks_t, st);
  return launch_kernel<T, 3>(mw, mx, p, blocks_n, blocks_t, st);
}

int check_shape(const tv_w4_args* a) {
  if (a->rows < 0 || a->n < 1 || a->group < 32 || a->group % 32 != 0 || a->k < a->group || a->k % a->group != 0)
    return TV_ERR_SHAPE;
  if (a->out_dtype != TV_BF16 && a->out_dtype != TV_F16) return TV_ERR_DTYPE;
  if (a->x_dtype != a->out_dtype && a->x_dtype != TV_E4M3) return TV_ERR_DTYPE;
  // the grid's token blocks, and the scale index by multiplication
  if (a->rows > 65535 * kMaxTokens || a->k > (1 << 20) || a->n > (1 << 27)) return TV_ERR_UNSUPPORTED;
  return TV_OK;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" {

int tv_w4_workspace_size(const tv_w4_args* a, size_t* bytes) {
  if (!a || !bytes) return TV_ERR_NULL;
  const int rc = check_shape(a);
  if (rc != TV_OK) return rc;
  *bytes = a->rows > 0 && !w4_rows_fit(a) && staged(a) ? (size_t)a->rows * padded_k(a->k) * 2 : 0;
  return TV_OK;
}

int tv_w4_linear(const tv_w4_args* a, void* stream) {
  if (!a) return TV_ERR_NULL;
  const int rc = check_shape(a);
  if (rc != TV_OK) return rc;
  if (a->rows == 0) return TV_OK;
  if (!a->x || !a->qweight || !a->scales || !a->out || (a->x_dtype == TV_E4M3 && !a->x_scale)) return TV_ERR_NULL;
  if (!aligned16(a->qweight) || a->q_sn % 4 != 0) return TV_ERR_ALIGN;
  if (a->q_sn < a->k / 8) return TV_ERR_SHAPE;
  if (w4_rows_fit(a)) return launch_w4_rows(a, static_cast<cudaStream_t>(stream));
  if (staged(a)) {
    size_t need = 0;
    tv_w4_workspace_size(a, &need);
    if (!a->workspace || a->workspace_bytes < need) return TV_ERR_WORKSPACE;
    if (!aligned16(a->workspace)) return TV_ERR_ALIGN;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->out_dtype == TV_BF16 ? launch_w4<__nv_bfloat16>(a, st) : launch_w4<__half>(a, st);
}

}  // extern "C"
