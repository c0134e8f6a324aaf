// int8_matmul.cu -- products of dynamically quantised activations with int8
// weights (W8A8): one scale per token, one per output channel, for one matrix
// or for the rows of several experts.  The reference's integer matrices are
// row-scaled int8 with f32 activations (HA:22-76); here both sides are int8.
//
//   s[r]      = fl32(max_c |x[r, c]| / 127),  q[r, c] = rne(fl32(x[r, c] / s[r]))
//   acc[r, n] = sum_k q[r, k] w[g, n, k]                (exact, int32)
//   out[r, n] = acc * s[r] * sw[g, n] + bias[g, n],  g the group of row r
//
// quant_kernel reads a row once into registers (DRAM-bound).  gemm_kernel runs
// tcgen05.mma kind::i8 with the weights as the A operand: M = 128 channels, N =
// up to 256 tokens, so that a decode step of one token fills the same 128 lanes
// as a prefill and streams the weights at full width; accumulators in TMEM,
// both operands staged by TMA (K-major rows of 128 bytes, 128-byte swizzle).
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "ffn_internal.h"
#include "rowops.cuh"
#include "tcgen05.cuh"

namespace ffn {
namespace i8 {

// The output of one sum: the same operations wherever it is formed.
__device__ __forceinline__ float product_value(int acc, float s, float sw, float bias) {
  return fmaf((float)acc * s, sw, bias);
}

// ---------------------------------------------------------------- quantise
struct QuantArgs {
  const void *x;
  size_t ld_x, ld_c;
  int8_t *codes;
  float *scales;
  const int32_t *n_rows;  // DEVICE count of rows in use, or NULL
  int rows;
  uint32_t cols, n_vec;
};

// The framework's gated activation (flash1017.rs:7539) of gate g and up u.  The fast
// division is within 2 steps, but gives 0 for a divisor above 2^126 (g below -87.3).
// What it drops there is below 1.1e-35, which no code shows unless the whole row is
// that small; such a row takes `SMALL`: from -64 down 1 + exp(-g) rounds to exp(-g),
// and the quotient is g exp(g).  (Taken for every value it cost 8192 x 2048 bf16 33
// us, 27 like this.)
constexpr float kSmallRow = 1e-28f;
template <bool SMALL>
__device__ __forceinline__ float swiglu10(float g, float u) {
  float silu;
  if (SMALL && g < -64.f) silu = g * expf(g);
  else silu = __fdividef(g, 1.0f + expf(-g));
  return fminf(silu, 10.0f) * fminf(fmaxf(u, -10.0f), 10.0f);
}

// Persistent, a row per CTA at a time; thread l holds the columns of pieces l, l +
// L, ... (16 in all) and has its pieces of the CTA's next row brought into shared
// memory meanwhile (STAGED; a third stage costs resident CTAs: 8192 x 4096 f32 30.4
// us, 28.0 with two).
constexpr int kQuantStages = 2;
template <typename T, int VEC, int NV, int MT, bool SWIGLU, bool STAGED>
__global__ void __launch_bounds__(MT) quant_kernel(const QuantArgs a) {
  constexpr int W = SWIGLU ? 2 : 1;  // gate and up
  __shared__ uint32_t s_red[2][32], s_small[32];
  extern __shared__ __align__(16) uint8_t s_dyn[];  // stages [kQuantStages][W][NV][threads] of 16 bytes
  pdl_enter();
  const uint32_t l = threadIdx.x, L = blockDim.x;
  const int lane = l & 31, warp = l >> 5, nw = L >> 5;
  const int rows = a.n_rows ? min(a.rows, *a.n_rows) : a.rows;
  uint4 *st = reinterpret_cast<uint4 *>(s_dyn) + l;
  auto fetch = [&](int stage, long long row) {
    if (row < rows) {
      const T *p = (const T *)a.x + (size_t)row * a.ld_x;
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (l + i * L < a.n_vec)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc::sa(st + ((stage * W + w) * NV + i) * L)),
                         "l"(p + (size_t)w * a.cols + (l + i * L) * VEC) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (STAGED)
    for (int q = 0; q < kQuantStages - 1; ++q) fetch(q, blockIdx.x + (long long)q * gridDim.x);
  int par = 0, stage = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, par ^= 1) {
    Raw<T, VEC> r[W][NV];
    if constexpr (STAGED) {
      fetch(stage == 0 ? kQuantStages - 1 : stage - 1, row + (long long)(kQuantStages - 1) * gridDim.x);
      asm volatile("cp.async.wait_group %0;" ::"n"(kQuantStages - 1) : "memory");
    }
    auto piece = [&](int w, int i) {
      if constexpr (STAGED) return *reinterpret_cast<const Raw<T, VEC> *>(st + ((stage * W + w) * NV + i) * L);
      else return load_raw<T, VEC>((const T *)a.x + (size_t)row * a.ld_x + (size_t)w * a.cols, l + i * L);
    };
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (l + i * L < a.n_vec) r[w][i] = piece(w, i);
    float f[SWIGLU ? NV : 1][VEC];
    // the activations of piece i, and the largest magnitude's bits
    auto gated = [&](auto small, const Raw<T, VEC> &gate, const Raw<T, VEC> &up, int i, uint32_t &m) {
      float u[VEC];
      unpack<T, VEC>(gate, f[i]);
      unpack<T, VEC>(up, u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        // the clamps would hide a gate or an up that is not finite
        const bool fin = isfinite(f[i][j]) && isfinite(u[j]);
        f[i][j] = swiglu10<decltype(small)::value>(f[i][j], u[j]);
        m = max(m, fin ? __float_as_uint(f[i][j]) & 0x7fffffffu : 0x7f800000u);
      }
    };
    auto cta_max = [&](uint32_t m, uint32_t *s) {
      m = __reduce_max_sync(0xffffffffu, m);
      if (nw > 1) {
        if (lane == 0) s[warp] = m;
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, lane < nw ? s[lane] : 0u);
      }
      return m;
    };
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (l + i * L >= a.n_vec) continue;
      if constexpr (SWIGLU) gated(std::false_type(), r[0][i], r[W - 1][i], i, m);
      else m = max(m, abs_bits<T, VEC>(r[0][i]));
    }
    m = cta_max(m, s_red[par]);
    if constexpr (SWIGLU) {
      if (m < __float_as_uint(kSmallRow)) {  // the whole CTA: m is the row's
        m = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (l + i * L < a.n_vec) gated(std::true_type(), piece(0, i), piece(W - 1, i), i, m);
        m = cta_max(m, s_small);
      }
    }
    stage = stage == kQuantStages - 1 ? 0 : stage + 1;
    const Int8Row sc = SWIGLU ? Int8Row(__uint_as_float(m)) : Int8Row::of_bits<T>(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (l + i * L >= a.n_vec) continue;
      float e[VEC];
      if (!SWIGLU) unpack<T, VEC>(r[0][i], e);
      store_codes<VEC>(a.codes + (size_t)row * a.ld_c + (size_t)(l + i * L) * VEC, SWIGLU ? f[SWIGLU ? i : 0] : e, sc);
    }
    if (l == 0) a.scales[row] = sc.scale();
  }
}

// ----------------------------------------------------------------- product
// Warp 0: TMA, one thread; warp 1: MMA, one thread; warps 2-5: epilogue.  The two
// single threads set the pace, so they count stages and phases instead of
// dividing.
constexpr int kMmaWarp = 1;
__host__ __device__ constexpr int threads_of(int mb) { return 64 + 128 * mb; }  // four epilogue warps a block of channels
constexpr int kM = 128;             // channels a block; a tile has one or two (MB)
constexpr int kKB = 128;            // K bytes (= values) a stage
constexpr int kABytes = kM * kKB;
constexpr int kMaxStages = 12;
constexpr int kSplitRows = 128;      // tokens a tile, at most, where K is split over a cluster
constexpr int kSmemMax = 224 * 1024;

struct GemmArgs {
  const int32_t *offsets;  // DEVICE [groups + 1] or NULL (one group of all rows)
  const float *xs, *ws, *bias;
  void *out;
  size_t ld_out;
  int rows, n, groups;
  int kt, kfull;  // 128-byte blocks of K, and those that are full
  int nt;      // tokens a tile, at most (a multiple of 16 up to 256)
  int sub;     // blocks of K a stage holds
  int stages;
  int cs;      // CTAs of the cluster, each a part of K
};

__device__ __forceinline__ uint32_t idesc_i8(int M, int N) {  // s32 += s8 * s8, both K-major
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc), "r"(0), "r"(0), "r"(0), "r"(0));
}
// Weights and tokens: tensor maps of 3-d boxes (128 bytes of K, rows, `sub` blocks
// of K), and of single blocks for a last one that is not full.
struct Maps {
  CUtensorMap w3, x3, w2, x2;
};
__device__ __forceinline__ void tma_3d(void *dst, const CUtensorMap *m, int y, int z, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(tc::sa(dst)), "l"(m), "r"(0), "r"(y), "r"(z), "r"(tc::sa(bar)) : "memory");
}
__device__ __forceinline__ void tma_2d(void *dst, const CUtensorMap *m, int x, int y, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(tc::sa(dst)), "l"(m), "r"(x), "r"(y), "r"(tc::sa(bar)) : "memory");
}
// Waits of this file: about two seconds, by the GPU's clock, after which `err`
// names the wait.
constexpr unsigned long long kWaitNs = 2000000000ull;
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool try_bar(uint64_t *b, uint32_t par) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok) : "r"(tc::sa(b)), "r"(par) : "memory");
  return ok != 0;
}
__device__ __noinline__ bool wait_bar_long(uint64_t *b, uint32_t par, int *err, int who) {
  unsigned long long end = 0;
  for (int i = 0;; ++i) {
    // test_wait returns at once (try_wait may sleep for as long as the hardware likes)
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(tc::sa(b)), "r"(par) : "memory");
    if (ok) return true;
    if ((i & 63) == 63) {
      if (err && *(volatile int *)err) return false;  // another role gave up
      const unsigned long long t = now_ns();
      if (end == 0) end = t + kWaitNs;
      else if (t > end) {
        if (err) atomicCAS_block(err, 0, who);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool wait_bar(uint64_t *b, uint32_t par, int *err, int who) {
  return try_bar(b, par) || wait_bar_long(b, par, err, who);
}
// for what completes by itself (copies, MMAs): not cut short by the others' errors
__device__ __forceinline__ void drain_bar(uint64_t *b, uint32_t par) {
  wait_bar(b, par, nullptr, 0);
}
__device__ __forceinline__ void tma_prefetch_l2(const CUtensorMap *m, int y, int z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(m), "r"(0), "r"(y), "r"(z) : "memory");
}
// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_peer(const void *p, uint32_t rank, int v) {
  uint32_t b;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(tc::sa(p)), "r"(rank));
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(b), "r"(v) : "memory");
}

// One tile: 128 MB channels of group g from channel c0, tokens [r0, r0 + nn).
struct Tile {
  int g, c0, r0, nn;
};
// s_pre[g]: token chunks of the groups before g.  Tiles run over the groups,
// inside a group over the channel blocks, inside a block over its token chunks,
// so CTAs that run together share the weights' block.
template <int MB>
__device__ __forceinline__ Tile tile_of(int t, const GemmArgs &a, const int *s_pre, const int *s_off, int ct) {
  int lo = 0, hi = a.groups;  // the last g with s_pre[g] * ct <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long long)s_pre[mid] * ct <= t) lo = mid; else hi = mid;
  }
  // skip empty groups: s_pre is equal there, the search ends on the last of them
  const int chunks = s_pre[lo + 1] - s_pre[lo], rel = t - s_pre[lo] * ct;
  const int first = s_off[2 * lo], n = s_off[2 * lo + 1];
  const int per = ((n + chunks - 1) / chunks + 15) & ~15;
  const int j = rel % chunks;
  Tile o;
  o.g = lo;
  o.c0 = rel / chunks * (MB * kM);
  o.r0 = first + j * per;
  o.nn = max(0, min(per, n - j * per));
  return o;
}

// MB = 2 halves the tokens' share of the traffic: with 128 x 256 tiles a dense
// prefill moves 48 KB a block of K from L2, 14 TB/s, which is what L2 gives; 256 x
// 256 tiles move 64 KB for twice the products.  Their two accumulators fill TMEM,
// so a tile's epilogue (eight warps) is not hidden behind the next one's MMAs.
template <typename T, int MB>
__global__ void __launch_bounds__(threads_of(MB), 1) gemm_kernel(const GemmArgs a, const __grid_constant__ Maps maps) {
  constexpr int kThreads = threads_of(MB), kBufs = MB == 1 ? 2 : 1, kWBytes = MB * kABytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], mma_done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_err, s_sum[threads_of(MB) / 32];
  __shared__ float s_xs[kSplitRows];
  uint8_t *smem = smem_raw + ((1024 - (tc::sa(smem_raw) & 1023)) & 1023);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  // a stage: sub blocks of weights, then sub blocks of tokens
  const int x_bytes = a.nt * kKB, stage_bytes = a.sub * (kWBytes + x_bytes);
  int *red = reinterpret_cast<int *>(smem + a.stages * stage_bytes);     // cs > 1: [cs][nt][128 / cs]
  const bool split = MB == 1 && a.cs > 1;
  int *s_off = red + (split ? kM * a.nt : 0);                          // [groups][first, count]
  int *s_pre = s_off + 2 * a.groups;                                      // [groups + 1]
  // Two accumulators; one where a cluster has a single tile.  It has at most 128
  // columns then (32 up to 32 tokens), and at least 175 KB of shared memory, so an
  // SM holds one such CTA, of whatever stream: clusters that waited for each
  // other's TMEM on two SMs would wait for good.  Other CTAs may share an SM (a K of
  // 256 in tiles of 256 tokens is 97 KB, but all of TMEM), and the allocation then
  // waits for the other's, of whatever stream.
  const int acc_cols = a.nt <= 16 ? 16 : 1 << (32 - __clz(a.nt - 1)), tmem_cols = split ? max(32, acc_cols) : 2 * acc_cols;
  const uint32_t rank = a.cs > 1 ? ctarank() : 0;
  const int ct = (a.n + MB * kM - 1) / (MB * kM);

  if (tid == 0) {
    s_err = 0;
    for (int s = 0; s < a.stages; ++s) { tc::bar_init(&full[s], 1); tc::bar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { tc::bar_init(&acc_full[b], 1); tc::bar_init(&acc_empty[b], 4 * MB); }
    tc::bar_init(&mma_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (a.kfull) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.w3) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.x3) : "memory");
    }
  }
  const int k_lo = split ? a.kt * (int)rank / a.cs : 0, k_hi = split ? a.kt * ((int)rank + 1) / a.cs : a.kt;
  const int tile0 = (int)(blockIdx.x / a.cs), tile_step = (int)(gridDim.x / a.cs);
  if (!a.offsets && warp == 0 && lane < a.stages && k_lo + lane * a.sub < min(k_hi, a.kfull)) {
    // one group: this CTA's first weights are known before the previous kernel
    // has finished; bring them into L2 (a hint, nothing is read from it yet)
    const int chunks = (a.rows + a.nt - 1) / a.nt;
    if (tile0 < chunks * ct)
      tma_prefetch_l2(&maps.w3, tile0 / chunks * MB * kM, k_lo + lane * a.sub);
  }
  pdl_enter();
  // Behind the wait for the previous kernel: whoever holds TMEM depends on nothing
  // but its own work.  A CTA that held it while it waited could hold what a CTA of
  // that previous kernel is still waiting for, itself or through another stream's.
  if (warp == kMmaWarp) tc::alloc(&s_tmem, tmem_cols);

  // token chunks of each group
  if (a.offsets) {
    const int per = (a.groups + kThreads - 1) / kThreads, g0 = min(tid * per, a.groups), g1 = min(g0 + per, a.groups);
    int sum = 0;
    for (int g = g0; g < g1; ++g) {
      // bounds from the GPU: kept inside the rows whatever they hold
      const int lo = min(max(a.offsets[g], 0), a.rows), hi = min(max(a.offsets[g + 1], lo), a.rows);
      s_off[2 * g] = lo;
      s_off[2 * g + 1] = hi - lo;
      s_pre[g] = sum;
      sum += (hi - lo + a.nt - 1) / a.nt;
    }
    int inc = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    int base = inc - sum;
    for (int w = 0; w < warp; ++w) base += s_sum[w];
    for (int g = g0; g < g1; ++g) s_pre[g] += base;
    if (tid == kThreads - 1) s_pre[a.groups] = base + sum;
  } else if (tid == 0) {
    s_off[0] = 0;
    s_off[1] = a.rows;
    s_pre[0] = 0;
    s_pre[1] = (a.rows + a.nt - 1) / a.nt;
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (split) cluster_arrive();  // waited for before the first sum goes to a peer
  const uint32_t tmem = s_tmem;
  const int n_tiles = s_pre[a.groups] * ct;

  if (warp == 0) {
    // -------------------------------------------------- TMA producer (one lane)
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0, used = 0;  // the stage, its phase, the stages ever used
      bool live = true;
      for (int t = tile0; t < n_tiles && live; t += tile_step) {
        const Tile o = tile_of<MB>(t, a, s_pre, s_off, ct);
        const int ch = o.g * a.n + o.c0;
        for (int k = k_lo; k < k_hi; k += a.sub) {
          if (!wait_bar(&empty[s], ph ^ 1, &s_err, 1)) { live = false; break; }
          uint8_t *sw = smem + s * stage_bytes, *sx = sw + a.sub * kWBytes;
          // One copy an operand for all blocks of a stage, as a single thread issues
          // them.  Blocks past the last full one read as zeros.
          const bool tail = a.kfull < a.kt && k + a.sub > a.kfull;
          const int n = tail ? min(a.sub, k_hi - k) : a.sub;
          tc::bar_arrive_tx(&full[s], n * (kWBytes + x_bytes));
          if (!tail) {
            tma_3d(sw, &maps.w3, ch, k, &full[s]);
            tma_3d(sx, &maps.x3, o.r0, k, &full[s]);
          } else {
            for (int q = 0; q < n; ++q) {
              tma_2d(sw + q * kWBytes, &maps.w2, (k + q) * kKB, ch, &full[s]);
              tma_2d(sx + q * x_bytes, &maps.x2, (k + q) * kKB, o.r0, &full[s]);
            }
          }
          used |= 1u << s;
          if (++s == a.stages) s = 0, ph ^= 1;
        }
      }
      // Every stage has been read before the CTA leaves: its copies have landed,
      // and no commit arrives in this shared memory any more.
      for (int i = 0; i < a.stages; ++i)
        if (used >> i & 1u) drain_bar(&empty[i], i < s ? ph : ph ^ 1);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // -------------------------------------------------- MMA issuer (one lane)
    if (elect_one()) {
      // Operand descriptors by addition: the start address (in 16 bytes) is their
      // low field and stays below its 14 bits.  elect.sync rather than a lane
      // number lets the compiler keep all of this in uniform registers, which is
      // where the instruction wants it.
      const uint64_t w0 = tc::desc_sw128(tc::sa(smem)), x0 = tc::desc_sw128(tc::sa(smem) + a.sub * kWBytes);
      uint64_t dw = w0, dx = x0;
      int s = 0, n = 0;
      uint32_t ph = 0;
      bool live = true;
      for (int t = tile0; t < n_tiles && live; t += tile_step, ++n) {
        const Tile o = tile_of<MB>(t, a, s_pre, s_off, ct);
        const uint32_t id = idesc_i8(kM, (o.nn + 15) & ~15);
        const int b = n % kBufs;
        if (!wait_bar(&acc_empty[b], ((n / kBufs) & 1) ^ 1, &s_err, 2)) break;
        tc::fence_after();
        const uint32_t d = tmem + b * acc_cols;
        uint32_t acc = 0;
        for (int k = k_lo; k < k_hi; k += a.sub) {
          const int nq = min(a.sub, k_hi - k);
          if (!wait_bar(&full[s], ph, &s_err, 3)) { live = false; break; }
          tc::fence_after();
          uint64_t qw = dw, qx = dx;
          for (int q = 0; q < nq; ++q, qw += kWBytes >> 4, qx += x_bytes >> 4) {
#pragma unroll
            for (int j = 0; j < kKB / 32; ++j, acc = 1)
#pragma unroll
              for (int mi = 0; mi < MB; ++mi)
                mma_i8(d + mi * acc_cols, qw + mi * (kABytes >> 4) + 2 * j, qx + 2 * j, id, acc);
          }
          tc::commit(&empty[s]);
          dw += stage_bytes >> 4, dx += stage_bytes >> 4;
          if (++s == a.stages) s = 0, ph ^= 1, dw = w0, dx = x0;
        }
        if (!live) break;
        tc::commit(&acc_full[b]);
      }
      tc::commit(&mma_done);  // every MMA has completed before TMEM is freed
      drain_bar(&mma_done, 0);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------- epilogue (4 MB warps)
    // the second four of MB = 2 take the second block of channels
    const int quarter = warp & 3, mi = (warp - kMmaWarp - 1) >> 2, cl = quarter * 32 + lane;
    int n = 0;
    if (split) cluster_wait();
    for (int t = tile0; t < n_tiles; t += tile_step, ++n) {
      const Tile o = tile_of<MB>(t, a, s_pre, s_off, ct);
      const int b = n % kBufs, ch = o.c0 + mi * kM + cl;
      const bool on = ch < a.n;
      // the scales, before the wait: column 32 i + lane's in xs[i].  Asked for in
      // the loop, their latency was a third of a tile with a short K (6144 x 1024 x
      // 4096 over 48 groups: 114 us, 48 us like this).
      float xs[8], sw = 0.f, bias = 0.f;
      if (!split) {
#pragma unroll
        for (int i = 0; i < 8; ++i) xs[i] = 32 * i + lane < o.nn ? a.xs[o.r0 + 32 * i + lane] : 0.f;
        if (on) {
          sw = a.ws[(size_t)o.g * a.n + ch];
          if (a.bias) bias = a.bias[(size_t)o.g * a.n + ch];
        }
      }
      const bool ok = __any_sync(0xffffffffu, lane == 0 && wait_bar(&acc_full[b], (n / kBufs) & 1, &s_err, 4));
      tc::fence_after();
      const uint32_t tl = tmem + (MB == 1 ? b : mi) * acc_cols + ((uint32_t)(32 * quarter) << 16);
      if (split) {
        // this CTA's part of K: lane cl's sums go to the CTA that owns the channel
        const int own = kM / a.cs, dst = cl / own;
        for (int c = 0; ok && c < o.nn; c += 16) {
          uint32_t v[16];
          tc::ld16(tl + c, v);
          tc::wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < o.nn) st_peer(red + ((int)rank * a.nt + c + j) * own + cl % own, dst, (int)v[j]);
        }
        break;  // one tile a cluster; the sums are added up below
      }
      T *out = reinterpret_cast<T *>(a.out) + (size_t)o.r0 * a.ld_out + ch;
      for (int c = 0; c < o.nn; c += 32) {
        uint32_t v[32];
        // (the columns from c + 16 are there if the tile has them: nt is a multiple
        // of 16, an accumulator a power of two)
        if (ok) {
          tc::ld16(tl + c, v);
          if (c + 16 < o.nn) tc::ld16(tl + c + 16, v + 16);
          tc::wait_ld();
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float s = __shfl_sync(0xffffffffu, xs[0], j);
          // a wait that ran out leaves NaN behind
          const float f = ok ? product_value((int)v[j], s, sw, bias) : __int_as_float(0x7fffffff);
          if (on && c + j < o.nn) *out = ToF32<T>::put(f);
          out += a.ld_out;
        }
#pragma unroll
        for (int i = 0; i < 7; ++i) xs[i] = xs[i + 1];
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::bar_arrive(&acc_empty[b]);
    }
  }
  if (split) {
    if (warp <= kMmaWarp) cluster_wait();
    // what the sums will be scaled by, loaded while they are on their way: a
    // thread keeps one channel of this CTA's own
    const Tile o = tile0 < n_tiles ? tile_of<MB>(tile0, a, s_pre, s_off, ct) : Tile{0, 0, 0, 0};
    const int own = kM / a.cs, c = tid % own, ch = o.c0 + (int)rank * own + c, step = kThreads / own;
    const bool on = ch < a.n && tid < step * own;
    const float sw = on ? a.ws[(size_t)o.g * a.n + ch] : 0.f;
    const float bias = on && a.bias ? a.bias[(size_t)o.g * a.n + ch] : 0.f;
    for (int i = tid; i < o.nn; i += kThreads) s_xs[i] = a.xs[o.r0 + i];
    __syncthreads();
    if (s_err && tid < a.cs) st_peer(&s_err, tid, 1);  // all CTAs of the cluster learn of it
    __syncwarp();
    cluster_sync();
    if (on) {
      T *out = reinterpret_cast<T *>(a.out) + (size_t)o.r0 * a.ld_out + ch;
      for (int r = tid / own; r < o.nn; r += step) {
        int acc = 0;
        for (int q = 0; q < a.cs; ++q) acc += red[(q * a.nt + r) * own + c];
        float f = product_value(acc, s_xs[r], sw, bias);
        if (s_err) f = __int_as_float(0x7fffffff);
        out[(size_t)r * a.ld_out] = ToF32<T>::put(f);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after();
    tc::dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------- few tokens, quantised in place
// A decode step of one or two tokens against one matrix: a single launch.  Every CTA
// quantises the tokens for itself (a few KB, L2 hits) while its warps' first
// weights are on the way; a warp then takes a channel at a time, 16 bytes a
// lane and load, and multiplies with dp4a.  Bound by the weights' bytes: 128 KB
// of loads in flight an SM.
constexpr int kFewRows = 2;
constexpr int kFewThreads = 512;
struct FewArgs {
  const void *x;
  size_t ld_x, ld_w, ld_out;
  const int8_t *w;
  const float *ws, *bias;
  void *out;
  int n, k, out_dtype;
  bool x16;  // x's rows can be read 16 bytes at a time
};
__host__ __device__ constexpr int few_pitch(int k) { return (k + 4095) / 4096 * 4096; }  // code bytes a token
constexpr int kFewCols = 16384;
static_assert(kFewRows * few_pitch(kFewCols) <= 47 * 1024, "the codes fit the launch default, less the static part");

// 16 weights from column 16 p of a row (zeros past k)
__device__ __forceinline__ uint4 few_piece(const int8_t *row, int p, int k) {
  if (16 * p + 16 <= k) return load_once(row + 16 * p);
  union { uint4 v; int8_t b[16]; } u;
  u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (16 * p + i < k) u.b[i] = row[16 * p + i];
  return u.v;
}

template <typename T, int R>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const FewArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) int8_t s_codes[];  // [R][few_pitch(k)]
  __shared__ uint32_t s_max[R][kFewThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kFewThreads / 32;
  const int pitch = few_pitch(a.k), step = gridDim.x * kWarps;
  int c = blockIdx.x * kWarps + warp;
  // while the previous kernel drains: a hint only, nothing is read
  if (c < a.n && lane * 128 < a.k)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + (size_t)c * a.ld_w + lane * 128));
  pdl_enter();
  uint4 w[8];
  auto load = [&](int ch, int base) {  // the 4096 bytes from column `base`
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = base / 16 + lane + 32 * j;
      w[j] = make_uint4(0, 0, 0, 0);
      if (ch < a.n && 16 * p < a.k) w[j] = few_piece(a.w + (size_t)ch * a.ld_w, p, a.k);
    }
  };

  // quantise: largest magnitudes, then codes.  The tokens are read before the
  // weights are asked for: behind 100 KB of weights an SM they came last.
  uint32_t m[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = 0;
    const T *x = (const T *)a.x + (size_t)r * a.ld_x;
    if (a.x16)
      for (int v = tid; v * VEC < a.k; v += kFewThreads) m[r] = max(m[r], abs_bits<T, VEC>(load_raw<T, VEC>(x, v)));
    else
      for (int v = tid; v < a.k; v += kFewThreads) m[r] = max(m[r], abs_bits<T, 1>(load_raw<T, 1>(x, v)));
    m[r] = __reduce_max_sync(0xffffffffu, m[r]);
    if (lane == 0) s_max[r][warp] = m[r];
  }
  load(c, 0);
  __syncthreads();
  float scale[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const Int8Row sc = Int8Row::of_bits<T>(__reduce_max_sync(0xffffffffu, lane < kWarps ? s_max[r][lane] : 0u));
    scale[r] = sc.scale();
    const T *x = (const T *)a.x + (size_t)r * a.ld_x;
    int8_t *q = s_codes + r * pitch;
    if (a.x16) {
      for (int v = tid; v * VEC < pitch; v += kFewThreads) {
        float e[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = 0.f;
        if (v * VEC < a.k) unpack<T, VEC>(load_raw<T, VEC>(x, v), e);
        store_codes<VEC>(q + v * VEC, e, sc);
      }
    } else {
      for (int v = tid; v < pitch; v += kFewThreads) {
        float e[1] = {0.f};
        if (v < a.k) unpack<T, 1>(load_raw<T, 1>(x, v), e);
        store_codes<1>(q + v, e, sc);
      }
    }
  }
  __syncthreads();

  for (; c < a.n; c += step) {
    int acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0;
    for (int base = 0; base < a.k; base += 4096) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (base + 512 * j >= a.k) break;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint4 q = *reinterpret_cast<const uint4 *>(s_codes + r * pitch + base + 16 * (lane + 32 * j));
          acc[r] = __dp4a((int)w[j].x, (int)q.x, acc[r]);
          acc[r] = __dp4a((int)w[j].y, (int)q.y, acc[r]);
          acc[r] = __dp4a((int)w[j].z, (int)q.z, acc[r]);
          acc[r] = __dp4a((int)w[j].w, (int)q.w, acc[r]);
        }
      }
      if (base + 4096 < a.k) load(c, base + 4096);
      else load(c + step, 0);
    }
    const float sw = a.ws[c], bias = a.bias ? a.bias[c] : 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[r]);
      const float f = product_value(sum, scale[r], sw, bias);
      if (lane == r) {
        const size_t at = (size_t)r * a.ld_out + c;
        if (a.out_dtype == FFN_B200_DT_F32) ((float *)a.out)[at] = f;
        else if (a.out_dtype == FFN_B200_DT_BF16) ((__nv_bfloat16 *)a.out)[at] = ToF32<__nv_bfloat16>::put(f);
        else ((__half *)a.out)[at] = ToF32<__half>::put(f);
      }
    }
  }
}

template <typename T>
int launch_few(const FewArgs &a, int rows, int sms, cudaStream_t st) {
  const int grid = std::min((a.n + kFewThreads / 32 - 1) / (kFewThreads / 32), sms * 4);
  const size_t smem = (size_t)rows * few_pitch(a.k);
#define FFN_GO(R) FFN_LAUNCH_PDL(FFN_B200_K_INT8_GEMM, st, "int8_linear", (few_kernel<T, R>), grid, kFewThreads, smem, a)
  if (rows == 1) FFN_GO(1);
  else FFN_GO(2);
#undef FFN_GO
  return 0;
}
bool few_fits(size_t rows, size_t k, size_t n_groups, const int32_t *offsets) {
  return rows <= (size_t)kFewRows && n_groups == 1 && !offsets && k <= (size_t)kFewCols;
}

// ------------------------------------------------------------------ launch
using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeFn)p;
  }();
  return fn;
}
// rows x k bytes at p, ld bytes apart, in boxes of 128 bytes x box_rows (x blocks,
// over the full blocks of 128 bytes alone); rows past the end, blocks past the
// last and bytes past k read as 0
int encode(CUtensorMap *m, const void *p, size_t rows, size_t k, size_t ld, int box_rows, int blocks) {
  const EncodeFn fn = encode_fn();
  if (!fn) return fail(FFN_B200_ECUDA, "int8_matmul: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dim[3] = {blocks ? (cuuint64_t)kKB : k, rows, k / kKB}, stride[2] = {ld, kKB};
  const cuuint32_t box[3] = {(cuuint32_t)kKB, (cuuint32_t)box_rows, (cuuint32_t)blocks}, es[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, blocks ? 3 : 2, const_cast<void *>(p), dim, stride, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FFN_B200_EINVAL, "int8_matmul: tensor map refused (code " + std::to_string((int)r) + ")");
  return 0;
}

template <typename T, int MB>
int launch_gemm(const GemmArgs &a, int grid, size_t smem, const Maps &maps, int dev, cudaStream_t st) {
  static bool attr[64] = {false};
  if (!attr[dev]) {
    FFN_CUDA_TRY(cudaFuncSetAttribute(gemm_kernel<T, MB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax));
    attr[dev] = true;
  }
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_allowed() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = a.cs;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads_of(MB));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = a.cs > 1 ? 2 : 1;
  prof_begin(FFN_B200_K_INT8_GEMM, st);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_kernel<T, MB>, a, maps);
  prof_end(FFN_B200_K_INT8_GEMM, st);
  note_launch();
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, "int8_matmul");
  }
  return 0;
}

// Checks a product and lays out its launch (p.grid 0: nothing to do).
struct GemmPlan {
  GemmArgs a;
  Maps maps;
  size_t smem;
  int grid, dev;
  int mb;  // blocks of 128 channels a tile
};
int plan_gemm(GemmPlan &p, size_t rows, size_t n, size_t k, size_t n_groups, const int32_t *offsets, const int8_t *x,
              size_t ld_x, const float *x_scales, const int8_t *w, size_t ld_w, const float *w_scales, const float *bias,
              int32_t dtype, void *out, size_t ld_out) {
  p.grid = 0;
  if (!dtype_ok(dtype)) return fail(FFN_B200_EINVAL, "int8_matmul: unknown dtype");
  if (n == 0 || k == 0 || k > 131072) return fail(FFN_B200_EUNSUP, "int8 product: n must be positive and k in 1..131072");
  if (n_groups == 0 || n_groups > 4096) return fail(FFN_B200_EINVAL, "int8_matmul: n_groups must be in 1..4096");
  if (n_groups > 1 && !offsets) return fail(FFN_B200_EINVAL, "int8_matmul: several groups need offsets");
  if (rows > (1u << 30) || n > (1u << 30) / n_groups) return fail(FFN_B200_EINVAL, "int8_matmul: too many rows");
  if (rows == 0) return 0;
  if (!x || !x_scales || !w || !w_scales || !out) return fail(FFN_B200_EINVAL, "int8_matmul: null pointer");
  if (((uintptr_t)x | (uintptr_t)w | ld_x | ld_w) % 16)
    return fail(FFN_B200_EINVAL, "int8_matmul: x, w and their row strides must be multiples of 16 bytes");
  if (ld_x < k || ld_w < k || (rows > 1 && ld_out < n)) return fail(FFN_B200_EINVAL, "int8_matmul: rows overlap");
  if ((uintptr_t)out % dtype_bytes(dtype) ||
      ((uintptr_t)x_scales | (uintptr_t)w_scales | (uintptr_t)bias | (uintptr_t)offsets) % 4)
    return fail(FFN_B200_EINVAL, "int8_matmul: out, scales and offsets must be aligned to their type");
  FFN_CUDA_TRY(cudaGetDevice(&p.dev));
  const int dev = p.dev;
  if (dev < 0 || dev >= 64) return fail(FFN_B200_EUNSUP, "int8_matmul: device index >= 64");
  const int sms = sm_count_of(dev);
  GemmArgs &a = p.a;
  a = GemmArgs{};
  a.offsets = offsets;
  a.xs = x_scales, a.ws = w_scales, a.bias = bias;
  a.out = out, a.ld_out = ld_out;
  a.rows = (int)rows, a.n = (int)n, a.groups = (int)n_groups;
  a.kt = (int)((k + kKB - 1) / kKB);
  a.kfull = (int)(k / kKB);
  const long long ct1 = (long long)((n + kM - 1) / kM), ct2 = (long long)((n + 2 * kM - 1) / (2 * kM));
  a.cs = 1;
  p.mb = 1;
  if (offsets) {
    // Groups: bound by the weights' bytes, so one chunk should hold a group: the
    // average and three deviations of an even routing.  Two blocks of channels only
    // for full tiles of 256 rows.  48 experts, K 2048, 4096 channels, f32 out, the
    // product alone: 128 rows each 92 us (tiles of 176 rows; 160 91, 128 97, 256 98;
    // two blocks of channels 93), 512 rows each 223 us (one block 241).
    // The average is over all rows given, also those behind the last group.
    const double avg = (double)rows / n_groups, want = avg + 3 * sqrt(avg);
    a.nt = want >= 256 ? 256 : std::max(16, ((int)ceil(want) + 15) / 16 * 16);
    if (want > 256 && n > (size_t)kM) p.mb = 2;
  } else {
    // One matrix: the cheapest tile by waves x blocks of K x time a block, in us as
    // measured at 4096 x 4096 (77 rows x 5120 x 2304: 9.5 us with 16 rows a tile,
    // 11.5 with 32, 12.9 with 48; 8192 rows: 101 us with 256 x 224 tiles, four full
    // waves, 106 with 256 x 256, 144 with 128 x 256).  K split over a cluster costs
    // 3.5 us more than it saves in blocks, and pays for few channels and a long K
    // (16 x 8192 x 1024: 7.9 us, 11.9 without).
    double best = 1e300;
    for (int nt = 16; nt <= 256; nt += 16) {
      const long long chunks = (long long)((rows + nt - 1) / nt), tiles = ct1 * chunks;
      const double n16 = (double)((((long long)rows + chunks - 1) / chunks + 15) / 16 * 16);
      const double block = std::min(0.10 + 0.0029 * n16, 0.30 + 0.00125 * n16);
      for (int cs = 1; cs <= 8; cs *= 2) {
        // (clusters that are sure to be resident at once)
        if (cs > 1 && (nt > kSplitRows || tiles * cs > sms * 3 / 4 || a.kt < 4 * cs)) break;
        const double us = cs == 1 ? ceil((double)tiles / sms) * a.kt * block : ceil((double)a.kt / cs) * block + 3.5 + 0.02 * n16;
        if (us < best) best = us, a.nt = nt, a.cs = cs, p.mb = 1;
      }
      if (nt >= 128 && n > (size_t)kM) {
        const double us = ceil((double)(ct2 * chunks) / sms) * (a.kt * (0.28 + 0.0021 * n16) + 1.0);
        if (us < best) best = us, a.nt = nt, a.cs = 1, p.mb = 2;
      }
      if ((size_t)nt >= rows) break;
    }
  }
  const long long ct = p.mb == 2 ? ct2 : ct1;
  // tiles at most: each group may end in a partial chunk
  const long long chunks = offsets ? std::min<long long>(rows, rows / a.nt + n_groups) : (rows + a.nt - 1) / a.nt;
  const long long tiles = ct * chunks;
  // (the kernel's tile numbers stay in 32 bits even where offsets are not ascending)
  if ((double)(rows / a.nt + 1) * (double)n_groups * (double)ct > 2147483647.0) return fail(FFN_B200_EINVAL, "int8_matmul: too many tiles");
  const size_t tail = (a.cs > 1 ? (size_t)kM * a.nt * 4 : 0) + (3 * n_groups + 1) * sizeof(int);
  const size_t block = (size_t)p.mb * kABytes + (size_t)a.nt * kKB, room = kSmemMax - 1024 - tail;
  // as many blocks a stage, up to 4, as leave three stages: each costs its threads
  // a wait and a commit (77 rows x 5120 x 2304 with its quantisation: 10.9 us, 14.8
  // with one; no effect on 8192 x 4096 x 4096),
  // and DRAM likes the rows' bytes together
  a.sub = 4;
  while (a.sub > 1 && (3 * a.sub * block > room || a.kt < 2 * a.sub * a.cs)) --a.sub;
  const size_t stage = a.sub * block;
  a.stages = (int)std::min<size_t>({room / stage, (size_t)kMaxStages, (size_t)std::max(2, a.kt)});
  if (a.stages < 2) return fail(FFN_B200_EUNSUP, "int8_matmul: too many groups for shared memory");
  p.smem = 1024 + a.stages * stage + tail;
  if (a.kfull) {
    if (int rc = encode(&p.maps.w3, w, n_groups * n, k, ld_w, p.mb * kM, a.sub)) return rc;
    if (int rc = encode(&p.maps.x3, x, rows, k, ld_x, a.nt, a.sub)) return rc;
  }
  if (a.kfull < a.kt) {
    if (int rc = encode(&p.maps.w2, w, n_groups * n, k, ld_w, p.mb * kM, 0)) return rc;
    if (int rc = encode(&p.maps.x2, x, rows, k, ld_x, a.nt, 0)) return rc;
  }
  p.grid = a.cs > 1 ? (int)tiles * a.cs : (int)std::min<long long>(tiles, sms);
  return 0;
}
template <typename T>
int run_gemm_as(const GemmPlan &p, cudaStream_t st) {
  return p.mb == 2 ? launch_gemm<T, 2>(p.a, p.grid, p.smem, p.maps, p.dev, st)
                   : launch_gemm<T, 1>(p.a, p.grid, p.smem, p.maps, p.dev, st);
}
int run_gemm(const GemmPlan &p, int32_t dtype, cudaStream_t st) {
  if (dtype == FFN_B200_DT_F32) return run_gemm_as<float>(p, st);
  if (dtype == FFN_B200_DT_BF16) return run_gemm_as<__nv_bfloat16>(p, st);
  return run_gemm_as<__half>(p, st);
}

template <typename T, int VEC, int MT, bool SWIGLU>
int launch_quant_as(QuantArgs &a, cudaStream_t st) {
  constexpr int NV = 16 / VEC;
  constexpr size_t kStage = (size_t)kQuantStages * (SWIGLU ? 2 : 1) * NV * 16;  // bytes a thread
  constexpr bool STAGED = VEC > 1 && kStage * MT <= (size_t)kSmemMax;
  const int threads = (int)((a.n_vec + 32 * NV - 1) / (32 * NV) * 32);
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(FFN_B200_EUNSUP, "quantize_int8: device index >= 64");
  const size_t smem = STAGED ? kStage * threads : 0;
  static bool attr[64] = {false};
  if (STAGED && !attr[dev]) {
    FFN_CUDA_TRY(cudaFuncSetAttribute(quant_kernel<T, VEC, NV, MT, SWIGLU, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(kStage * MT)));
    attr[dev] = true;
  }
  static int resident[64][MT / 32 + 1] = {{0}};
  int &per_sm = resident[dev][threads / 32];
  if (per_sm == 0) {
    int n = 0;
    FFN_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, quant_kernel<T, VEC, NV, MT, SWIGLU, STAGED>, threads, smem));
    per_sm = std::max(1, n);
  }
  const int grid = (int)std::min<long long>(a.rows, (long long)sm_count_of(dev) * per_sm);
  FFN_LAUNCH_PDL(FFN_B200_K_INT8_QUANT, st, "quantize_int8", (quant_kernel<T, VEC, NV, MT, SWIGLU, STAGED>), grid, threads, smem, a);
  return 0;
}
template <typename T, int VEC, bool SWIGLU>
int launch_quant(QuantArgs &a, cudaStream_t st) {
  a.n_vec = a.cols / VEC;
  if (a.cols <= 4096) return launch_quant_as<T, VEC, 256, SWIGLU>(a, st);
  if (a.cols <= 8192) return launch_quant_as<T, VEC, 512, SWIGLU>(a, st);
  return launch_quant_as<T, VEC, 1024, SWIGLU>(a, st);
}
template <typename T, int VEC>
int launch_quant_act(QuantArgs &a, int act, cudaStream_t st) {
  return act == FFN_B200_ACT_SWIGLU ? launch_quant<T, VEC, true>(a, st) : launch_quant<T, VEC, false>(a, st);
}

}  // namespace i8
}  // namespace ffn

using namespace ffn;

extern "C" {

int ffn_b200_quantize_int8(size_t rows, size_t cols, int32_t dtype, const void *x, size_t ld_x, int32_t act,
                           const int32_t *n_rows, int8_t *codes, size_t ld_codes, float *scales, void *stream) {
  using namespace ffn::i8;
  if (!dtype_ok(dtype)) return fail(FFN_B200_EINVAL, "quantize_int8: unknown dtype");
  if (act != FFN_B200_ACT_NONE && act != FFN_B200_ACT_SWIGLU) return fail(FFN_B200_EINVAL, "quantize_int8: unknown act");
  if (cols == 0 || cols > 16384) return fail(FFN_B200_EUNSUP, "quantize_int8: cols must be in 1..16384");
  if (rows > 0x7fffffffu) return fail(FFN_B200_EINVAL, "quantize_int8: too many rows");
  if (rows == 0) return 0;
  if (!x || !codes || !scales) return fail(FFN_B200_EINVAL, "quantize_int8: null pointer");
  const size_t width = act == FFN_B200_ACT_SWIGLU ? 2 * cols : cols, es = dtype_bytes(dtype);
  if (rows > 1 && (ld_x < width || ld_codes < cols)) return fail(FFN_B200_EINVAL, "quantize_int8: rows overlap");
  if ((uintptr_t)x % es || ((uintptr_t)scales | (uintptr_t)n_rows) % 4)
    return fail(FFN_B200_EINVAL, "quantize_int8: rows, scales and n_rows must be aligned to their type");
  QuantArgs a{};
  a.x = x, a.ld_x = ld_x, a.codes = codes, a.ld_c = ld_codes, a.scales = scales, a.n_rows = n_rows;
  a.rows = (int)rows, a.cols = (uint32_t)cols;
  const bool v16 = cols * es % 16 == 0 && rows16(x, ld_x, es) && (((uintptr_t)codes | ld_codes) & 7) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FFN_B200_DT_F32) return v16 ? launch_quant_act<float, 4>(a, act, st) : launch_quant_act<float, 1>(a, act, st);
  if (dtype == FFN_B200_DT_BF16)
    return v16 ? launch_quant_act<__nv_bfloat16, 8>(a, act, st) : launch_quant_act<__nv_bfloat16, 1>(a, act, st);
  return v16 ? launch_quant_act<__half, 8>(a, act, st) : launch_quant_act<__half, 1>(a, act, st);
}

int ffn_b200_int8_matmul(size_t rows, size_t n, size_t k, size_t n_groups, const int32_t *offsets, const int8_t *x,
                         size_t ld_x, const float *x_scales, const int8_t *w, size_t ld_w, const float *w_scales,
                         const float *bias, int32_t dtype, void *out, size_t ld_out, void *stream) {
  using namespace ffn::i8;
  GemmPlan p{};
  if (int rc = plan_gemm(p, rows, n, k, n_groups, offsets, x, ld_x, x_scales, w, ld_w, w_scales, bias, dtype, out, ld_out))
    return rc;
  return p.grid ? run_gemm(p, dtype, (cudaStream_t)stream) : 0;
}

size_t ffn_b200_int8_linear_ws_bytes(size_t rows, size_t k, size_t n_groups, const int32_t *offsets) {
  if (ffn::i8::few_fits(rows, k, n_groups, offsets)) return 0;
  return rows * ((k + 15) / 16 * 16 + sizeof(float));
}

int ffn_b200_int8_linear(size_t rows, size_t n, size_t k, size_t n_groups, const int32_t *offsets, int32_t x_dtype,
                         const void *x, size_t ld_x, const int8_t *w, size_t ld_w, const float *w_scales, const float *bias,
                         int32_t dtype, void *out, size_t ld_out, void *ws, size_t ws_bytes, void *stream) {
  using namespace ffn::i8;
  if (!dtype_ok(x_dtype) || !dtype_ok(dtype)) return fail(FFN_B200_EINVAL, "int8_linear: unknown dtype");
  if (n == 0 || k == 0 || k > 16384) return fail(FFN_B200_EUNSUP, "int8_linear: n must be positive and k in 1..16384");
  if (!few_fits(rows, k, n_groups, offsets)) {
    const size_t ld = (k + 15) / 16 * 16;
    if (rows > (1u << 30)) return fail(FFN_B200_EINVAL, "int8_linear: too many rows");
    if (rows && (!ws || (uintptr_t)ws % 16)) return fail(FFN_B200_EINVAL, "int8_linear: the workspace is null or misaligned");
    if (ws_bytes < rows * (ld + sizeof(float))) return fail(FFN_B200_ENOSPC, "int8_linear: workspace too small");
    int8_t *codes = (int8_t *)ws;
    float *scales = (float *)(codes + rows * ld);
    GemmPlan p{};
    if (int rc = plan_gemm(p, rows, n, k, n_groups, offsets, codes, ld, scales, w, ld_w, w_scales, bias, dtype, out, ld_out))
      return rc;
    // rows behind the last group's are in no product: not quantised either
    if (int rc = ffn_b200_quantize_int8(rows, k, x_dtype, x, ld_x, FFN_B200_ACT_NONE, offsets ? offsets + n_groups : nullptr,
                                        codes, ld, scales, stream))
      return rc;
    return p.grid ? run_gemm(p, dtype, (cudaStream_t)stream) : 0;
  }
  if (rows == 0) return 0;
  if (!x || !w || !w_scales || !out) return fail(FFN_B200_EINVAL, "int8_linear: null pointer");
  if (((uintptr_t)w | ld_w) % 16) return fail(FFN_B200_EINVAL, "int8_linear: w and its row stride must be multiples of 16 bytes");
  if (n > (1u << 30)) return fail(FFN_B200_EINVAL, "int8_linear: too many channels");
  if (ld_w < k || (rows > 1 && (ld_out < n || ld_x < k))) return fail(FFN_B200_EINVAL, "int8_linear: rows overlap");
  const size_t es = dtype_bytes(x_dtype);
  if ((uintptr_t)x % es || (uintptr_t)out % dtype_bytes(dtype) || ((uintptr_t)w_scales | (uintptr_t)bias) % 4)
    return fail(FFN_B200_EINVAL, "int8_linear: rows and scales must be aligned to their type");
  FewArgs a{};
  a.x = x, a.ld_x = ld_x, a.w = w, a.ld_w = ld_w, a.ws = w_scales, a.bias = bias;
  a.out = out, a.ld_out = ld_out, a.out_dtype = dtype;
  a.n = (int)n, a.k = (int)k;
  a.x16 = k * es % 16 == 0 && rows16(x, ld_x, es);
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  const int sms = sm_count_of(dev);
  cudaStream_t st = (cudaStream_t)stream;
  if (x_dtype == FFN_B200_DT_F32) return launch_few<float>(a, (int)rows, sms, st);
  if (x_dtype == FFN_B200_DT_BF16) return launch_few<__nv_bfloat16>(a, (int)rows, sms, st);
  return launch_few<__half>(a, (int)rows, sms, st);
}

}  // extern "C"
