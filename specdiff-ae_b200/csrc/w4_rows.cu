// Up to 8 rows times 4-bit weights with group scales (one token, a draft's
// frontier): the weights go from HBM through registers into mma.sync, with no
// shared memory, tensor memory or barrier on their way.
//
// One CTA per SM, so that x is staged once an SM; its four teams of four warps
// take 16 weight rows at a time (M of m16n8k16; the rows of x are its N),
// dealt out SM by SM so that none has more than one unit above another.  A
// team's warps split k, 128 at a time: lane t of quad g loads the 16 bytes, 32
// weights, of k = 32 t .. 32 t + 31 of rows g and g + 8.  The MMA sums over k
// whatever its order, so the four lanes' k need not interleave as the
// fragment's do, only match x's: x lies in shared memory as 16-byte units of
// 8 k in the order ((128-k block, 8 k of 32), row, t), and a B fragment of two
// MMAs is one conflict-free 16-byte load.  Eight blocks of 128 k are in flight
// per warp: each block's registers are loaded anew, eight blocks ahead, as soon
// as it is used.  A team's sums meet in shared memory and are added in order.
//
// The weights are rounded to the 16-bit type as the kernel for more rows has to,
// although a block's scale could meet its fp32 sums instead where a group covers
// it: a token alone and the same token in a tree then differ in 0.04 % of the
// outputs (bf16, 4096 x 4096, alone and among 65) where 40 % did with unrounded
// weights here, and a draft's verification has to see the model that decodes.
// Leaving the rounding out gave 16.6 -> 16.5 us in bf16 and 20.1 -> 18.8 in fp16
// at 8 x 28672 x 4096.
//
// The first eight blocks come to L2 by one bulk request a row while the kernel
// before this one ends (16.3 -> 15.1 us at one row x 28672 x 4096, 18.0 -> 16.6 at
// 8); requests further ahead, all along the way, were slower (18.2 and 19.7).
//
// One row x 28672 x 4096 takes 15.1 us, 8 rows 16.6 (9.3 at the measured HBM
// rate), and no pipe is at its limit: about 140 instructions a warp for 2048
// weights, 72 of them the unpacking, are 7 us of every scheduler's 16.6, HBM runs
// at 56 %.  3 us go to the start and the first round trip, the rest to waits for
// loads that eight blocks in flight do not cover.  The uneven last round is not
// it: 28416 rows, three units for every team, take 16.1 us.
//
// That is with the four scales of a batch in one load: group 128, k a multiple of
// 2048.  Elsewhere each lane loads the scale of its 32 k by itself: 8 rows x 28672
// x 4096 take 28.5 us at group 64 and 27.9 at 256, one row x 4096 x 11008 takes
// 15.4 (10240: 8.0).
//
// Whole units a warp (no split of k) took 18.9 us at 8 x 28672 x 4096, but 10.4 for
// 7.7 at 8 x 6144 x 4096; teams of eight 19.5 and 8.1.  Two tiles of N (16 rows)
// took 10.2 us for the tcgen05 kernel's 10.5 at 6144 x 4096 and 26.1 for 22.4 at
// 28672 x 4096 (group 128), so that takes over at 9.
#include <cuda_fp8.h>

#include <type_traits>

#include "w4.cuh"

namespace tv {
namespace {

using namespace w4;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kTeam = 4;                // warps that share 16 weight rows
constexpr int kTeams = kWarps / kTeam;
constexpr int kM = 16;                  // weight rows per unit
constexpr int kBlockK = 128;
constexpr int kBatch = 4;               // blocks of a batch; two batches are in flight
constexpr int kMaxRows = 8;             // N of m16n8k16
constexpr int kMaxSmem = 220 * 1024;

struct Params {
  const void* x;
  int64_t x_sm;
  const float* x_scale;
  const uint32_t* q;
  int64_t q_sn;
  const void* s;
  int64_t s_sn;
  void* out;
  int64_t o_sm;
  int rows, n, k, blocks, units;
  uint32_t magic;
};

// Eight consecutive values of a row as 16-bit pairs; zeros past k.
template <typename X, typename T>
__device__ __forceinline__ uint4 load8(const X* p, bool in, bool vec) {
  uint4 o = make_uint4(0, 0, 0, 0);
  if (!in) return o;
  if constexpr (std::is_same<X, T>::value) {
    if (vec) return *reinterpret_cast<const uint4*>(p);
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t) * reinterpret_cast<const uint16_t*>(p + 2 * i) |
             (uint32_t) * reinterpret_cast<const uint16_t*>(p + 2 * i + 1) << 16;
  } else {
    alignas(8) X b[8];
    if (vec) {
      *reinterpret_cast<uint2*>(b) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = p[i];
    }
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Elem<T>::pack2(static_cast<float>(b[2 * i]), static_cast<float>(b[2 * i + 1]));
  }
  return o;
}

// X: type of x (T or e4m3).  FOUR: group 128 with whole batches, the four
// scales of one in one load.
template <typename T, typename X, bool FOUR>
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* xs = reinterpret_cast<uint4*>(smem);
  float* red = reinterpret_cast<float*>(smem + (size_t)p.blocks * kBlockK * 2 * p.rows);   // [2][warps][8][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // a warp's run of 128-k blocks, none where there are fewer than warps
  const int part = warp % kTeam, team = warp / kTeam;
  const int lo = p.blocks * part / kTeam, hi = p.blocks * (part + 1) / kTeam;
  const int stride = gridDim.x * kTeams;

  struct Batch {
    uint4 w[kBatch][2];
    uint32_t s[kBatch][2];      // a block's scales; with FOUR [0][h], [1][h] are the batch's four
  };
  // What is loaded next: block b of unit's rows 16 unit + g and + 8; rows past
  // the end repeat the last one (not stored), k past the end weighs nothing.
  struct Ahead {
    int unit, b;
    const uint32_t *q0, *q1;
    const T *s0, *s1;
  } ahead{(int)(blockIdx.x + gridDim.x * team), lo, nullptr, nullptr, nullptr, nullptr};
  auto at_unit = [&] {
    const int64_t n0 = min(ahead.unit * kM + g, p.n - 1), n1 = min(ahead.unit * kM + g + 8, p.n - 1);
    ahead.q0 = p.q + n0 * p.q_sn + t * 4;
    ahead.q1 = p.q + n1 * p.q_sn + t * 4;
    ahead.s0 = static_cast<const T*>(p.s) + n0 * p.s_sn;
    ahead.s1 = static_cast<const T*>(p.s) + n1 * p.s_sn;
  };
  auto words4 = [](const uint32_t* at, uint4& v) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
  };
  auto scale1 = [](const T* at, uint32_t& v) {
    asm volatile("{\n\t.reg .u16 v;\n\tld.global.nc.u16 v, [%1];\n\tcvt.u32.u16 %0, v;\n\t}" : "=r"(v) : "l"(at));
  };
  auto load_block = [&](int i, Batch& o) {
    const int b = ahead.b + i;
    if (FOUR || (b < hi && (b * 4 + t) * 32 < p.k)) {
      words4(ahead.q0 + b * (kBlockK / 8), o.w[i][0]);
      words4(ahead.q1 + b * (kBlockK / 8), o.w[i][1]);
      if (!FOUR) {
        const uint32_t u = (uint32_t)(b * 4 + t), j = p.magic ? __umulhi(u, p.magic) : u;
        scale1(ahead.s0 + j, o.s[i][0]);
        scale1(ahead.s1 + j, o.s[i][1]);
      }
    } else {
      o.s[i][0] = o.s[i][1] = 0;
    }
  };
  auto load_four = [&](Batch& o) {
    asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(o.s[0][0]), "=r"(o.s[1][0]) : "l"(ahead.s0 + ahead.b));
    asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(o.s[0][1]), "=r"(o.s[1][1]) : "l"(ahead.s1 + ahead.b));
  };
  auto advance = [&] {
    ahead.b += kBatch;
    if (ahead.b >= hi) {
      ahead.b = lo;
      ahead.unit += stride;
      at_unit();
    }
  };
  grid_next();
  // the first weights may come to L2 before the predecessor's end: what it
  // still writes is seen there all the same
  if (ahead.unit < p.units && lane < kM && lo < hi) {
    const int bytes = min(min(lo + 2 * kBatch, hi) * kBlockK, p.k) / 2 - lo * (kBlockK / 2);
    const uint32_t* at = p.q + (int64_t)min(ahead.unit * kM + lane, p.n - 1) * p.q_sn + lo * (kBlockK / 8);
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(bytes) : "memory");
  }
  grid_wait();
  Batch ping{}, pong{};
  int unit = ahead.unit, b = lo;
  at_unit();
  auto fill = [&](Batch& o) {
    if (ahead.unit < p.units) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) load_block(i, o);
      if (FOUR) load_four(o);
      advance();
    }
  };
  fill(ping);
  fill(pong);

  // x into shared memory while the first weights are on their way
  {
    const X* x = static_cast<const X*>(p.x);
    const int chunks = p.blocks * (kBlockK / 8);
    const int total = p.rows * chunks;
    const bool vec = (reinterpret_cast<uintptr_t>(x) % (8 * sizeof(X))) == 0 && (p.rows == 1 || p.x_sm % 8 == 0);
    // unit e of the layout: 8 k of (block and 8 of 32, row, t)
#pragma unroll 4
    for (int e = threadIdx.x; e < total; e += kThreads) {
      const int kj = (e >> 2) / p.rows, r = (e >> 2) - kj * p.rows;
      const int c = (kj >> 2) * 16 + (e & 3) * 4 + (kj & 3);     // its k is 8 c
      xs[e] = load8<X, T>(x + (int64_t)r * p.x_sm + c * 8, c * 8 < p.k, vec);
    }
  }
  __syncthreads();

  // this lane's row of x (column of B) in xs; past the last row, whose sums
  // are not stored, the last
  const int xrow = min(g, p.rows - 1) * 4;
  int turn = 0;
  float acc[4] = {};
  // One batch of the present unit, each block's registers refilled two batches
  // ahead as soon as it is used; at the unit's end the warps' sums.  False once
  // there is no unit left.
  auto step = [&](Batch& now) {
    const bool last = b + kBatch >= hi, more = ahead.unit < p.units;
    const uint4* xb = xs + b * 16 * p.rows + t;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (FOUR || b + i < hi) {
        Unpack<T> u0, u1;
        u0.scale(FOUR ? __byte_perm(now.s[i >> 1][0], 0, i & 1 ? 0x3232 : 0x1010) : now.s[i][0] * 0x10001u);
        u1.scale(FOUR ? __byte_perm(now.s[i >> 1][1], 0, i & 1 ? 0x3232 : 0x1010) : now.s[i][1] * 0x10001u);
        const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&now.w[i][0]);
        const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&now.w[i][1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0[4], a1[4];
          u0.word(w0[j], a0);
          u1.word(w1[j], a1);
          const uint32_t f0[4] = {a0[0], a1[0], a0[1], a1[1]}, f1[4] = {a0[2], a1[2], a0[3], a1[3]};
          const uint4 v = xb[(i * 4 + j) * p.rows * 4 + xrow];
          Mma<T>::run(acc, f0, v.x, v.y);
          Mma<T>::run(acc, f1, v.z, v.w);
        }
      }
      if (more) load_block(i, now);
    }
    if (more) {
      if (FOUR) load_four(now);
      advance();
    }
    b += kBatch;
    if (!last) return true;
    // accumulator i of a lane: weight row g + 8 (i / 2), x row 2 t + i % 2
    float* mine = red + (turn * kWarps + warp) * (kM * kMaxRows);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mine[(2 * t + (i & 1)) * kM + g + 8 * (i >> 1)] = acc[i];
      acc[i] = 0.f;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(kTeam * 32) : "memory");
    const float* ours = red + (turn * kWarps + team * kTeam) * (kM * kMaxRows);
    const int e = part * 32 + lane, n = unit * kM + e % kM;
    static_assert(kTeam * 32 == kM * kMaxRows, "a thread of the team per sum");
    if (e / kM < p.rows && n < p.n) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kTeam; ++w) sum += ours[w * (kM * kMaxRows) + e];
      sum *= Unpack<T>::unscale();
      if (p.x_scale) sum *= __ldg(p.x_scale + e / kM);
      static_cast<T*>(p.out)[(int64_t)(e / kM) * p.o_sm + n] = Elem<T>::from_f(sum);
    }
    turn ^= 1;      // the other half is free: every warp of the team has passed the barrier after reading it
    b = lo;
    unit += stride;
    return unit < p.units;
  };
  if (unit < p.units)
    while (step(ping) && step(pong)) {
    }
}

size_t smem_bytes(const tv_w4_args* a) {
  const size_t blocks = (a->k + kBlockK - 1) / kBlockK;
  return blocks * kBlockK * 2 * a->rows + 2 * kWarps * kM * kMaxRows * sizeof(float);
}

template <typename T, typename X, bool FOUR>
int start(const Params& p, int grid, size_t smem, cudaStream_t st) {
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(w4_rows_kernel<T, X, FOUR>), (int)smem);
  if (rc != TV_OK) return rc;
  return launch_early(w4_rows_kernel<T, X, FOUR>, dim3((unsigned)grid), kThreads, smem, 0, st, p);
}

template <typename T, typename X>
int launch(const tv_w4_args* a, Params p, size_t smem, cudaStream_t st) {
  const int grid = p.units < kNumSMs ? p.units : kNumSMs;
  const bool four = a->group == kBlockK && p.blocks % (kTeam * kBatch) == 0 && a->s_sn % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(a->scales) % 8 == 0;
  return four ? start<T, X, true>(p, grid, smem, st) : start<T, X, false>(p, grid, smem, st);
}

template <typename T>
int dispatch(const tv_w4_args* a, const Params& p, size_t smem, cudaStream_t st) {
  return a->x_dtype == TV_E4M3 ? launch<T, __nv_fp8_e4m3>(a, p, smem, st) : launch<T, T>(a, p, smem, st);
}

}  // namespace

bool w4_rows_fit(const tv_w4_args* a) { return a->rows <= kMaxRows && smem_bytes(a) <= kMaxSmem; }

int launch_w4_rows(const tv_w4_args* a, cudaStream_t st) {
  Params p{};
  p.x = a->x;
  p.x_sm = a->x_sm;
  p.x_scale = a->x_dtype == TV_E4M3 ? a->x_scale : nullptr;
  p.q = static_cast<const uint32_t*>(a->qweight);
  p.q_sn = a->q_sn;
  p.s = a->scales;
  p.s_sn = a->s_sn;
  p.out = a->out;
  p.o_sm = a->o_sm;
  p.rows = a->rows;
  p.n = a->n;
  p.k = a->k;
  p.blocks = (a->k + kBlockK - 1) / kBlockK;
  p.units = (a->n + kM - 1) / kM;
  p.magic = group_magic(a->group);
  const size_t smem = smem_bytes(a);
  return a->out_dtype == TV_BF16 ? dispatch<__nv_bfloat16>(a, p, smem, st) : dispatch<__half>(a, p, smem, st);
}

}  // namespace tv
