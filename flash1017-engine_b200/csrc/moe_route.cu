// moe_route.cu -- routed pairs sorted by expert and back, as callable
// operators: the layer's grouping and combine (flash1017.rs:8088-8099,
// 8267-8326) for activation rows of any type, with their gradients.
//
//   sort      pairs (t, k) of idx [T, K] ordered by expert, by pair number
//             inside an expert: pos[t, k] = row, src[row] = pair, offsets
//   permute   xs[pos[t, k]] = x[t]
//   combine   out[t] = residual[t] + sum_k w[t, k] y[pos[t, k]]
//   gradients dx[t] = sum_k dxs[pos[t, k]] (combine without weights),
//             dy[pos[t, k]] = w[t, k] dout[t], dw[t, k] = <dout[t], y[pos[t, k]]>
//
// Every sum runs in f32 in a fixed order and no kernel uses atomics, so results
// do not change from call to call.
#include <algorithm>

#include "ffn_internal.h"
#include "rowops.cuh"

namespace ffn {
namespace route {

// ------------------------------------------------------------------- sort
// A stable counting sort in one launch: one thread-block cluster, each warp a
// contiguous segment of the pairs.  A warp ranks 32 pairs at a time (the lanes
// with the same expert, found by a ballot per bit of the expert number, in lane
// order), so the order inside an expert is the pair order.  match.any finds the
// same lanes in one instruction, but its latency was most of the kernel's time.
// Counts per (segment, expert) sit in shared memory; the CTAs of the cluster read
// each other's totals over distributed shared memory, which saves the second and
// third launch and the workspace that a grid-wide sort would need.  Bound by
// latency, not by bytes: 8 bytes a pair.  src is scattered by the same kernel
// (49152 pairs: 9.5 us; 10.0 with a second kernel that wrote it from pos).
constexpr int kSortThreads = 1024;
constexpr int kSortCluster = 16;    // most CTAs of a cluster (8 are portable)
constexpr int kSortBatch = 8;
constexpr int kSortCounts = 32768;  // (segments per CTA) x (local experts): 128 KB of counters

struct SortArgs {
  const int32_t *idx;
  int n_pairs, e_begin, n_local;
  int segs;     // segments (warps that rank) per CTA
  int per_seg;  // pairs per segment, a multiple of 32
  int32_t *offsets, *pos, *src;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int peer_int(const int *p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), b;
  int v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(b));
  return v;
}

// the lanes whose v (below 2^bits) is this lane's
__device__ __forceinline__ uint32_t same_lanes(uint32_t v, int bits) {
  uint32_t m = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = v >> b & 1u;
    const uint32_t set = __ballot_sync(0xffffffffu, one);
    m &= one ? set : ~set;
  }
  return m;
}

__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const SortArgs a) {
  extern __shared__ int s_cnt[];  // [segs][n_local], then [n_local] totals, then [n_local] first rows
  __shared__ int s_warp[32];
  __shared__ int s_carry;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), nrank = cluster_size();
  int *tot = s_cnt + a.segs * a.n_local, *off = tot + a.n_local;
  // pass 1: counts per segment.  kSortBatch groups of ids are asked for before the
  // first is ranked: one at a time, their latency was most of the time.
  const long long s0 = ((long long)rank * a.segs + warp) * a.per_seg;
  const int p0 = (int)min(s0, (long long)a.n_pairs), p1 = (int)min(s0 + a.per_seg, (long long)a.n_pairs);
  int *mine = s_cnt + warp * a.n_local;
  auto ids = [&](int p, int (&e)[kSortBatch]) {
#pragma unroll
    for (int i = 0; i < kSortBatch; ++i) {
      e[i] = -1;
      if (p + 32 * i + lane < p1) {
        // unsigned: ids below e_begin, and the top-k step's "no candidate"
        // 0x7fffffff, fall outside like those at or above the range's end
        const uint32_t r = (uint32_t)a.idx[p + 32 * i + lane] - (uint32_t)a.e_begin;
        if (r < (uint32_t)a.n_local) e[i] = (int)r;
      }
    }
  };
  int e[kSortBatch], rk[kSortBatch];  // rk: the pair's number inside its expert and segment
  const int bits = 32 - __clz(a.n_local);
  if (warp < a.segs) ids(p0, e);
  for (int i = tid; i < a.segs * a.n_local; i += kSortThreads) s_cnt[i] = 0;
  __syncthreads();
  if (warp < a.segs) {
    for (int p = p0; p < p1; p += 32 * kSortBatch) {
      if (p > p0) ids(p, e);
#pragma unroll
      for (int i = 0; i < kSortBatch; ++i) {
        if (p + 32 * i >= p1) break;
        const uint32_t same = same_lanes(e[i] < 0 ? a.n_local : e[i], bits);
        const int base = e[i] >= 0 ? mine[e[i]] : 0;
        rk[i] = base + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e[i] >= 0 && lane == __ffs(same) - 1) mine[e[i]] = base + __popc(same);
        __syncwarp();
      }
    }
  }
  __syncthreads();
  // counts -> exclusive prefix over this CTA's segments; totals
  for (int x = tid; x < a.n_local; x += kSortThreads) {
    int run = 0;
#pragma unroll 8
    for (int s = 0; s < a.segs; ++s) {
      const int c = s_cnt[s * a.n_local + x];
      s_cnt[s * a.n_local + x] = run;
      run += c;
    }
    tot[x] = run;
  }
  __syncthreads();  // the cluster barrier is .aligned: whole warps arrive
  cluster_arrive();
  cluster_wait();
  // exclusive prefix over the experts of the cluster's totals; the pairs of
  // lower-ranked CTAs come first inside an expert
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int x0 = 0; x0 < a.n_local; x0 += kSortThreads) {
    const int x = x0 + tid;
    int all = 0, before = 0;
    if (x < a.n_local) {
      int c[kSortCluster];
#pragma unroll
      for (uint32_t r = 0; r < kSortCluster; ++r) c[r] = r < nrank ? peer_int(tot + x, r) : 0;
#pragma unroll
      for (uint32_t r = 0; r < kSortCluster; ++r) {
        all += c[r];
        if (r < rank) before += c[r];
      }
    }
    int inc = all;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      int v = s_warp[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      s_warp[lane] = v;
    }
    __syncthreads();
    const int first = s_carry + (warp ? s_warp[warp - 1] : 0) + inc - all;
    if (x < a.n_local) {
      off[x] = first + before;
      if (rank == 0) a.offsets[x] = first;
    }
    __syncthreads();
    if (tid == 0) s_carry += s_warp[31];
    __syncthreads();
  }
  const int total = s_carry;
  if (rank == 0 && tid == 0) a.offsets[a.n_local] = total;
  cluster_arrive();  // the reads of the peers' totals are done; waited for at the end

  // pass 2: rows.  One batch (up to 256 pairs a segment) is still in registers with
  // its numbers; longer segments are ranked again.
  if (warp < a.segs) {
    const bool kept = a.per_seg <= 32 * kSortBatch;
    for (int p = p0; p < p1; p += 32 * kSortBatch) {
      if (!kept) ids(p, e);
#pragma unroll
      for (int i = 0; i < kSortBatch; ++i) {
        if (p + 32 * i >= p1) break;
        const int at = p + 32 * i + lane, first = e[i] >= 0 ? mine[e[i]] : 0;
        if (!kept) {
          const uint32_t same = same_lanes(e[i] < 0 ? a.n_local : e[i], bits);
          rk[i] = __popc(same & ((1u << lane) - 1u));
          __syncwarp();
          if (e[i] >= 0 && lane == __ffs(same) - 1) mine[e[i]] = first + __popc(same);
          __syncwarp();
        }
        const int row = e[i] >= 0 ? off[e[i]] + first + rk[i] : -1;
        if (at < p1) {
          if (a.pos) a.pos[at] = row;
          if (a.src && row >= 0) a.src[row] = at;
        }
      }
    }
  }
  if (a.src)  // rows behind the last local pair
    for (long long r = total + (long long)rank * kSortThreads + tid; r < a.n_pairs; r += (long long)nrank * kSortThreads)
      a.src[r] = -1;
  __syncwarp();
  cluster_wait();
}

// Work layout of the row kernels: `tpt` threads (a power of two, 32 .. 256) share
// a token, a CTA of 256 holds 256 / tpt tokens; a warp works on one token, its
// lanes hold the token's pos and weights (choice k in lane k % 32) and hand them
// round by shuffles.  The next token's are loaded while this one's rows move, so
// that the chain of two DRAM latencies (pos, then rows) is not paid per token.

// ------------------------------------------------- permute (rows of bytes)
// blockIdx.y cuts long rows into segments of tpt * kPieces pieces; each piece is
// read once and written to the token's rows.  DRAM-bound by the written rows
// (stores alone reach 6.7 TB/s on this GPU).
constexpr int kPieces = 4;
template <int BYTES>
__global__ void __launch_bounds__(256) permute_kernel(const uint8_t *x, size_t ld_x, const int32_t *pos, uint8_t *out,
                                                      size_t ld_out, int n_tok, int top_k, uint32_t n_vec,
                                                      uint32_t out_rows, const float *x_scale, float *out_scale, int tpt) {
  using R = typename RawOf<BYTES>::type;
  pdl_enter();
  const int l = threadIdx.x & (tpt - 1), per = 256 / tpt, lane = threadIdx.x & 31;
  const uint32_t v0 = blockIdx.y * (uint32_t)(tpt * kPieces) + l;
  const long long step = (long long)gridDim.x * per;
  long long t = (long long)blockIdx.x * per + threadIdx.x / tpt;
  auto lookup = [&](long long tok, int k) { return tok < n_tok && k < top_k ? pos[(size_t)tok * top_k + k] : -1; };
  int32_t next = lookup(t, lane);
  for (; t < n_tok; t += step) {
    int32_t pl = next;
    next = lookup(t + step, lane);
    R r[kPieces];
    const R *xr = reinterpret_cast<const R *>(x + (size_t)t * ld_x);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (v0 + i * tpt < n_vec) r[i] = xr[v0 + i * tpt];
    const float s = x_scale && v0 == 0 ? x_scale[t] : 0.f;
    for (int k = 0; k < top_k; ++k) {
      if (k && (k & 31) == 0) pl = lookup(t, k + lane);
      const uint32_t p = (uint32_t)__shfl_sync(0xffffffffu, pl, k & 31);
      if (p >= out_rows) continue;
      R *o = reinterpret_cast<R *>(out + (size_t)p * ld_out);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (v0 + i * tpt < n_vec) o[v0 + i * tpt] = r[i];
      if (x_scale && v0 == 0) out_scale[p] = s;
    }
  }
}

// ----------------------------------------------------------------- combine
// A thread's piece of AHEAD routed rows is loaded before the first is used.
// DRAM-bound by the experts' rows, so what counts is loads on their way: with 6
// ahead 64 registers are enough and 1024 threads an SM fit (8 ahead and 768
// threads: 24576 rows of 4096 bf16 and a residual take 61 us, like this 52).
// Single elements (VEC 1) go four to a thread, so that looking a row up is not
// most of the instructions (8192 x 6 x 4095 bf16: 501 us with one, 165 us).
template <typename T, int VEC, int AHEAD>
__global__ void __launch_bounds__(256, AHEAD > 6 ? 3 : 4) combine_rows_kernel(const T *y, size_t ld_y, uint32_t y_rows, const int32_t *pos,
                                                              const float *w, const T *residual, size_t ld_r, T *out,
                                                              size_t ld_o, int n_tok, int top_k, uint32_t n_vec, int tpt) {
  constexpr int P = VEC == 1 ? 4 : 1;
  pdl_enter();
  const int l = threadIdx.x & (tpt - 1), per = 256 / tpt, lane = threadIdx.x & 31;
  const uint32_t v0 = blockIdx.y * (uint32_t)(tpt * P) + l;
  const long long step = (long long)gridDim.x * per;
  long long t = (long long)blockIdx.x * per + threadIdx.x / tpt;
  auto lookup = [&](long long tok, int k) { return tok < n_tok && k < top_k ? pos[(size_t)tok * top_k + k] : -1; };
  auto weight = [&](long long tok, int k) { return w && tok < n_tok && k < top_k ? w[(size_t)tok * top_k + k] : 1.f; };
  int32_t next = lookup(t, lane);
  float next_w = weight(t, lane);
  for (; t < n_tok; t += step) {
    int32_t pl = next;
    float wl = next_w;
    next = lookup(t + step, lane);
    next_w = weight(t + step, lane);
    Raw<T, VEC> rr[P] = {};
    if (residual)
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (v0 + i * tpt < n_vec) rr[i] = load_raw<T, VEC>(residual + (size_t)t * ld_r, v0 + i * tpt);
    float acc[P][VEC];
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[i][j] = 0.f;
    for (int k0 = 0; k0 < top_k; k0 += AHEAD) {
      if (k0 && (k0 & 31) == 0) pl = lookup(t, k0 + lane), wl = weight(t, k0 + lane);
      Raw<T, VEC> r[AHEAD][P];
      uint32_t use = 0;
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const uint32_t p = (uint32_t)__shfl_sync(0xffffffffu, pl, (k0 + q) & 31);
        if (k0 + q < top_k && p < y_rows) {
          use |= 1u << q;
          const T *row = y + (size_t)p * ld_y;
#pragma unroll
          for (int i = 0; i < P; ++i)
            if (v0 + i * tpt < n_vec) r[q][i] = load_raw<T, VEC>(row, v0 + i * tpt);
        }
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const float f = __shfl_sync(0xffffffffu, wl, (k0 + q) & 31);
        if (use >> q & 1u)
#pragma unroll
          for (int i = 0; i < P; ++i)
            if (v0 + i * tpt < n_vec) {
              float e[VEC];
              unpack<T, VEC>(r[q][i], e);
#pragma unroll
              for (int j = 0; j < VEC; ++j) acc[i][j] = fmaf(f, e[j], acc[i][j]);
            }
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (v0 + i * tpt >= n_vec) continue;
      if (residual) {
        float e[VEC];
        unpack<T, VEC>(rr[i], e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[i][j] += e[j];
      }
      store_vec<T, VEC>(out + (size_t)t * ld_o, v0 + i * tpt, acc[i]);
    }
  }
}

// ------------------------------------------------------- combine, backward
// TPT threads (one warp, or the CTA) a token: the token's gradient row is read
// once per kBack choices (again from L1), each choice's row of y once, each row
// of dy written once; the kBack dot products are reduced together.  kBack = 8
// takes 128 registers, two CTAs an SM (4096 tokens x 6 x 4096 bf16: 93 us; 4: 79
// us).
constexpr int kBack = 4;
template <typename T, int VEC, int TPT>
__global__ void __launch_bounds__(256, 3) combine_bwd_kernel(const T *dout, size_t ld_d, const T *y, size_t ld_y,
                                                          uint32_t y_rows, const int32_t *pos, const float *w, T *dy,
                                                          size_t ld_dy, float *dw, int n_tok, int top_k, uint32_t n_vec) {
  constexpr int kTok = 256 / TPT, P = VEC == 1 ? 4 : 1;  // single elements four to a thread
  __shared__ float s_red[2][8][kBack];
  pdl_enter();
  const int l = threadIdx.x % TPT, lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * kTok;
  long long t = (long long)blockIdx.x * kTok + threadIdx.x / TPT;
  auto lookup = [&](long long tok, int k) { return tok < n_tok && k < top_k ? pos[(size_t)tok * top_k + k] : -1; };
  auto weight = [&](long long tok, int k) { return w && tok < n_tok && k < top_k ? w[(size_t)tok * top_k + k] : 1.f; };
  int32_t next = lookup(t, lane);
  float next_w = weight(t, lane);
  int par = 0;
  for (; t < n_tok; t += step) {
    int32_t pl = next;
    float wl = next_w;
    next = lookup(t + step, lane);
    next_w = weight(t + step, lane);
    const T *drow = dout + (size_t)t * ld_d;
    for (int k0 = 0; k0 < top_k; k0 += kBack, par ^= 1) {
      if (k0 && (k0 & 31) == 0) pl = lookup(t, k0 + lane), wl = weight(t, k0 + lane);
      uint32_t p[kBack];
      float f[kBack], dot[kBack];
#pragma unroll
      for (int q = 0; q < kBack; ++q) {
        p[q] = (uint32_t)__shfl_sync(0xffffffffu, pl, (k0 + q) & 31);
        if (k0 + q >= top_k || p[q] >= y_rows) p[q] = 0xffffffffu;
        f[q] = __shfl_sync(0xffffffffu, wl, (k0 + q) & 31);
        dot[q] = 0.f;
      }
      for (uint32_t v = l; v < n_vec; v += TPT * P) {
        Raw<T, VEC> r[kBack][P], rd[P] = {};
        if (dw) {
#pragma unroll
          for (int q = 0; q < kBack; ++q)
            if (p[q] != 0xffffffffu)
#pragma unroll
              for (int i = 0; i < P; ++i)
                if (v + i * TPT < n_vec) r[q][i] = load_raw<T, VEC>(y + (size_t)p[q] * ld_y, v + i * TPT);
        }
#pragma unroll
        for (int i = 0; i < P; ++i)
          if (v + i * TPT < n_vec) rd[i] = load_raw<T, VEC>(drow, v + i * TPT);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if (v + i * TPT >= n_vec) continue;
          float d[VEC];
          unpack<T, VEC>(rd[i], d);
          if (dy) {
#pragma unroll
            for (int q = 0; q < kBack; ++q)
              if (p[q] != 0xffffffffu) {
                float e[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) e[j] = f[q] * d[j];
                store_vec<T, VEC>(dy + (size_t)p[q] * ld_dy, v + i * TPT, e);
              }
          }
          if (dw) {
#pragma unroll
            for (int q = 0; q < kBack; ++q)
              if (p[q] != 0xffffffffu) {
                float e[VEC];
                unpack<T, VEC>(r[q][i], e);
#pragma unroll
                for (int j = 0; j < VEC; ++j) dot[q] = fmaf(d[j], e[j], dot[q]);
              }
          }
        }
      }
      if (dw) {
#pragma unroll
        for (int q = 0; q < kBack; ++q) dot[q] = warp_sum(dot[q]);
        if (TPT > 32) {
          if (lane == 0)
#pragma unroll
            for (int q = 0; q < kBack; ++q) s_red[par][threadIdx.x >> 5][q] = dot[q];
          __syncthreads();  // par: the next sums go elsewhere, so one barrier a round
          if (threadIdx.x < kBack && k0 + (int)threadIdx.x < top_k) {
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < 8; ++g) s += s_red[par][g][threadIdx.x];
            dw[(size_t)t * top_k + k0 + threadIdx.x] = s;
          }
        } else {
#pragma unroll
          for (int q = 0; q < kBack; ++q)
            if (lane == q && k0 + q < top_k) dw[(size_t)t * top_k + k0 + q] = dot[q];
        }
      }
    }
  }
}

// ------------------------------------------------------------------ launch
// CTAs for the work, `resident` an SM at most (each then takes several tokens and
// looks the next one up in time).
int grid_of(long long ctas, int resident) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  return (int)std::max(1LL, std::min<long long>(ctas, (long long)sm_count_of(dev) * resident));
}
// Threads a token: the most of 256, 128, 64, 32 that leaves at most a tenth of
// them without a piece in the row's last segment.
int threads_per_token(uint32_t n_vec, int pieces) {
  for (int t = 256; t > 32; t /= 2) {
    const uint64_t seg = (n_vec + (uint64_t)t * pieces - 1) / ((uint64_t)t * pieces);
    if (seg * t * pieces * 10 <= (uint64_t)n_vec * 11) return t;
  }
  return 32;
}

template <int BYTES>
int launch_permute(const void *x, size_t ld_x, const int32_t *pos, void *out, size_t ld_out, size_t n_tok, size_t top_k,
                   size_t row_bytes, size_t out_rows, const float *xs, float *os, cudaStream_t st) {
  const uint32_t n_vec = (uint32_t)(row_bytes / BYTES);
  int tpt = threads_per_token(n_vec, 1);
  const uint32_t seg = (n_vec + tpt * kPieces - 1) / (tpt * kPieces);
  if (seg > 65535) return fail(FFN_B200_EUNSUP, "moe_permute: row too long for its alignment");
  const dim3 grid(grid_of((long long)(n_tok + 256 / tpt - 1) / (256 / tpt), std::max<int>(1, 32 / seg)), seg);
  FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "permute_kernel", (permute_kernel<BYTES>), grid, 256, 0, (const uint8_t *)x, ld_x, pos,
                 (uint8_t *)out, ld_out, (int)n_tok, (int)top_k, n_vec, (uint32_t)out_rows, xs, os, tpt);
  return 0;
}

template <typename T, int VEC, int AHEAD>
int launch_combine_as(const void *y, size_t ld_y, size_t y_rows, const int32_t *pos, const float *w, const void *res,
                      size_t ld_r, void *out, size_t ld_o, size_t n_tok, size_t top_k, size_t cols, cudaStream_t st) {
  const uint32_t n_vec = (uint32_t)(cols / VEC);
  constexpr int P = VEC == 1 ? 4 : 1;
  const int tpt = threads_per_token(n_vec, P);
  const uint32_t seg = (n_vec + tpt * P - 1) / (tpt * P);
  if (seg > 65535) return fail(FFN_B200_EUNSUP, "moe_combine: row too long for its alignment");
  const dim3 grid(grid_of((long long)(n_tok + 256 / tpt - 1) / (256 / tpt), 32), seg);
  FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "combine_rows_kernel", (combine_rows_kernel<T, VEC, AHEAD>), grid, 256, 0, (const T *)y,
                 ld_y, (uint32_t)y_rows, pos, w, (const T *)res, ld_r, (T *)out, ld_o, (int)n_tok, (int)top_k, n_vec, tpt);
  return 0;
}
// rows loaded ahead: all of a token's up to 8; a batch never straddles the 32
// choices that a warp's lanes hold
template <typename T, int VEC>
int launch_combine_rows(const void *y, size_t ld_y, size_t y_rows, const int32_t *pos, const float *w, const void *res,
                        size_t ld_r, void *out, size_t ld_o, size_t n_tok, size_t top_k, size_t cols, cudaStream_t st) {
#define FFN_CALL(A) launch_combine_as<T, VEC, A>(y, ld_y, y_rows, pos, w, res, ld_r, out, ld_o, n_tok, top_k, cols, st)
  if (top_k <= 4) return FFN_CALL(4);
  if (top_k <= 6) return FFN_CALL(6);
  return FFN_CALL(8);
#undef FFN_CALL
}

template <typename T, int VEC>
int launch_combine_bwd(const void *dout, size_t ld_d, const void *y, size_t ld_y, size_t y_rows, const int32_t *pos,
                       const float *w, void *dy, size_t ld_dy, float *dw, size_t n_tok, size_t top_k, size_t cols,
                       cudaStream_t st) {
  const uint32_t n_vec = (uint32_t)(cols / VEC);
  // a warp a token up to 4 pieces a lane; a CTA a token above
  if (n_vec <= 128) {
    const int grid = grid_of((long long)(n_tok + 7) / 8, 3);
    FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "combine_bwd_kernel", (combine_bwd_kernel<T, VEC, 32>), grid, 256, 0,
                   (const T *)dout, ld_d, (const T *)y, ld_y, (uint32_t)y_rows, pos, w, (T *)dy, ld_dy, dw, (int)n_tok,
                   (int)top_k, n_vec);
  } else {
    const int grid = grid_of((long long)n_tok, 3);
    FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "combine_bwd_kernel", (combine_bwd_kernel<T, VEC, 256>), grid, 256, 0,
                   (const T *)dout, ld_d, (const T *)y, ld_y, (uint32_t)y_rows, pos, w, (T *)dy, ld_dy, dw, (int)n_tok,
                   (int)top_k, n_vec);
  }
  return 0;
}

// Checks shared by permute, combine and combine_bwd.
int check_pairs(const char *what, size_t n_tok, size_t top_k, size_t rows) {
  if (top_k == 0 || top_k > 4096) return fail(FFN_B200_EINVAL, std::string(what) + ": top_k must be in 1..4096");
  if (n_tok > (1u << 30) / top_k) return fail(FFN_B200_EINVAL, std::string(what) + ": too many routed pairs");
  if (rows > 0x7fffffffu) return fail(FFN_B200_EINVAL, std::string(what) + ": too many rows");
  return 0;
}

}  // namespace route
}  // namespace ffn

using namespace ffn;

extern "C" {

int ffn_b200_moe_sort(size_t n_tok, size_t top_k, const int32_t *idx, int32_t expert_begin, int32_t expert_end,
                      int32_t *offsets, int32_t *pos, int32_t *src, void *stream) {
  using namespace ffn::route;
  if (int rc = check_pairs("moe_sort", n_tok, top_k, 0)) return rc;
  if (!offsets || (n_tok && !idx)) return fail(FFN_B200_EINVAL, "moe_sort: null pointer");
  if (((uintptr_t)idx | (uintptr_t)offsets | (uintptr_t)pos | (uintptr_t)src) % 4)
    return fail(FFN_B200_EINVAL, "moe_sort: arrays must be 4-byte aligned");
  if (expert_begin < 0 || expert_end <= expert_begin || expert_end - expert_begin > 4096)
    return fail(FFN_B200_EINVAL, "moe_sort: the expert range must be 1..4096 experts from expert_begin >= 0");
  cudaStream_t st = (cudaStream_t)stream;
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(FFN_B200_EUNSUP, "moe_sort: device index >= 64");
  SortArgs a{};
  a.idx = idx;
  a.n_pairs = (int)(n_tok * top_k);
  a.e_begin = expert_begin;
  a.n_local = expert_end - expert_begin;
  a.offsets = offsets;
  a.pos = pos;
  a.src = src;
  // One CTA up to 512 pairs (384 experts: 4.5 us for 384 pairs, but 7.3 us for 2046
  // against 4.5 us with the cluster).
  // Above 8192 pairs 16 CTAs (49152 pairs: 12.0 us with 8, 9.5 us), where this
  // GPU can hold such a cluster.
  static int widest[64] = {0};
  if (!widest[dev]) {
    FFN_CUDA_TRY(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (kSortCounts + 2 * 4096) * (int)sizeof(int)));
    FFN_CUDA_TRY(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchAttribute ca;
    ca.id = cudaLaunchAttributeClusterDimension;
    ca.val.clusterDim.x = kSortCluster;
    ca.val.clusterDim.y = ca.val.clusterDim.z = 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(kSortCluster);
    c.blockDim = dim3(kSortThreads);
    c.dynamicSmemBytes = (kSortCounts + 2 * 4096) * sizeof(int);
    c.attrs = &ca;
    c.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, sort_kernel, &c) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    widest[dev] = n > 0 ? kSortCluster : 8;
  }
  const int nclu = a.n_pairs <= 512 ? 1 : a.n_pairs <= 8192 ? 8 : widest[dev];
  const int groups = (a.n_pairs + 31) / 32, per_cta = (groups + nclu - 1) / nclu;
  a.segs = std::max(1, std::min({kSortThreads / 32, kSortCounts / a.n_local, per_cta}));
  a.per_seg = std::max(1, (per_cta + a.segs - 1) / a.segs) * 32;
  const size_t smem = ((size_t)a.segs * a.n_local + 2 * (size_t)a.n_local) * sizeof(int);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_allowed() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = nclu;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(nclu);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  prof_begin(FFN_B200_K_ROUTE, st);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sort_kernel, a);
  prof_end(FFN_B200_K_ROUTE, st);
  note_launch();
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, "moe_sort");
  }
  return 0;
}

int ffn_b200_moe_permute(size_t n_tok, size_t top_k, size_t row_bytes, const void *x, size_t ld_x, const int32_t *pos,
                         size_t out_rows, void *out, size_t ld_out, const float *x_scale, float *out_scale,
                         void *stream) {
  using namespace ffn::route;
  if (int rc = check_pairs("moe_permute", n_tok, top_k, out_rows)) return rc;
  if (n_tok == 0 || out_rows == 0) return 0;
  if (!x || !pos || !out) return fail(FFN_B200_EINVAL, "moe_permute: null pointer");
  if ((x_scale == nullptr) != (out_scale == nullptr))
    return fail(FFN_B200_EINVAL, "moe_permute: x_scale and out_scale go together");
  if (((uintptr_t)pos | (uintptr_t)x_scale | (uintptr_t)out_scale) % 4)
    return fail(FFN_B200_EINVAL, "moe_permute: pos and scales must be 4-byte aligned");
  if (row_bytes == 0 || row_bytes > (1u << 30)) return fail(FFN_B200_EINVAL, "moe_permute: bad row size");
  if ((n_tok > 1 && ld_x < row_bytes) || (out_rows > 1 && ld_out < row_bytes))
    return fail(FFN_B200_EINVAL, "moe_permute: rows overlap");
  const uintptr_t all = (uintptr_t)x | (uintptr_t)out | ld_x | ld_out | row_bytes;
  cudaStream_t st = (cudaStream_t)stream;
  if (all % 16 == 0) return launch_permute<16>(x, ld_x, pos, out, ld_out, n_tok, top_k, row_bytes, out_rows, x_scale, out_scale, st);
  if (all % 4 == 0) return launch_permute<4>(x, ld_x, pos, out, ld_out, n_tok, top_k, row_bytes, out_rows, x_scale, out_scale, st);
  if (all % 2 == 0) return launch_permute<2>(x, ld_x, pos, out, ld_out, n_tok, top_k, row_bytes, out_rows, x_scale, out_scale, st);
  return launch_permute<1>(x, ld_x, pos, out, ld_out, n_tok, top_k, row_bytes, out_rows, x_scale, out_scale, st);
}

int ffn_b200_moe_combine(size_t n_tok, size_t top_k, size_t cols, int32_t dtype, const void *y, size_t ld_y,
                         size_t y_rows, const int32_t *pos, const float *w, const void *residual, size_t ld_res, void *out,
                         size_t ld_out, void *stream) {
  using namespace ffn::route;
  if (int rc = check_pairs("moe_combine", n_tok, top_k, y_rows)) return rc;
  if (!dtype_ok(dtype)) return fail(FFN_B200_EINVAL, "moe_combine: unknown dtype");
  if (cols == 0 || cols > (1u << 28)) return fail(FFN_B200_EINVAL, "moe_combine: bad cols");
  if (n_tok == 0) return 0;
  if ((!y && y_rows) || !pos || !out) return fail(FFN_B200_EINVAL, "moe_combine: null pointer");
  if ((y_rows > 1 && ld_y < cols) || (n_tok > 1 && (ld_out < cols || (residual && ld_res < cols))))
    return fail(FFN_B200_EINVAL, "moe_combine: rows overlap");
  const size_t es = dtype_bytes(dtype);
  if (((uintptr_t)y | (uintptr_t)residual | (uintptr_t)out) % es)
    return fail(FFN_B200_EINVAL, "moe_combine: rows must be aligned to their type");
  if (((uintptr_t)pos | (uintptr_t)w) % 4) return fail(FFN_B200_EINVAL, "moe_combine: pos and w must be 4-byte aligned");
  const bool v16 = cols * es % 16 == 0 && rows16(y, ld_y, es) && rows16(out, ld_out, es) && rows16(residual, ld_res, es);
  cudaStream_t st = (cudaStream_t)stream;
#define FFN_CALL(T, V) launch_combine_rows<T, V>(y, ld_y, y_rows, pos, w, residual, ld_res, out, ld_out, n_tok, top_k, cols, st)
  if (dtype == FFN_B200_DT_F32) return v16 ? FFN_CALL(float, 4) : FFN_CALL(float, 1);
  if (dtype == FFN_B200_DT_BF16) return v16 ? FFN_CALL(__nv_bfloat16, 8) : FFN_CALL(__nv_bfloat16, 1);
  return v16 ? FFN_CALL(__half, 8) : FFN_CALL(__half, 1);
#undef FFN_CALL
}

int ffn_b200_moe_combine_bwd(size_t n_tok, size_t top_k, size_t cols, int32_t dtype, const void *dout, size_t ld_dout,
                             const void *y, size_t ld_y, size_t y_rows, const int32_t *pos, const float *w, void *dy,
                             size_t ld_dy, float *dw, void *stream) {
  using namespace ffn::route;
  if (int rc = check_pairs("moe_combine_bwd", n_tok, top_k, y_rows)) return rc;
  if (!dtype_ok(dtype)) return fail(FFN_B200_EINVAL, "moe_combine_bwd: unknown dtype");
  if (cols == 0 || cols > (1u << 28)) return fail(FFN_B200_EINVAL, "moe_combine_bwd: bad cols");
  if (n_tok == 0 || (!dy && !dw)) return 0;
  if (!dout || !pos || (dw && !y && y_rows)) return fail(FFN_B200_EINVAL, "moe_combine_bwd: null pointer");
  if ((n_tok > 1 && ld_dout < cols) || (y_rows > 1 && ((dw && ld_y < cols) || (dy && ld_dy < cols))))
    return fail(FFN_B200_EINVAL, "moe_combine_bwd: rows overlap");
  const size_t es = dtype_bytes(dtype);
  if (((uintptr_t)y | (uintptr_t)dout | (uintptr_t)dy) % es)
    return fail(FFN_B200_EINVAL, "moe_combine_bwd: rows must be aligned to their type");
  if (((uintptr_t)pos | (uintptr_t)w | (uintptr_t)dw) % 4)
    return fail(FFN_B200_EINVAL, "moe_combine_bwd: pos, w and dw must be 4-byte aligned");
  const bool v16 = cols * es % 16 == 0 && rows16(dw ? y : nullptr, ld_y, es) && rows16(dout, ld_dout, es) && rows16(dy, ld_dy, es);
  cudaStream_t st = (cudaStream_t)stream;
#define FFN_CALL(T, V) launch_combine_bwd<T, V>(dout, ld_dout, y, ld_y, y_rows, pos, w, dy, ld_dy, dw, n_tok, top_k, cols, st)
  if (dtype == FFN_B200_DT_F32) return v16 ? FFN_CALL(float, 4) : FFN_CALL(float, 1);
  if (dtype == FFN_B200_DT_BF16) return v16 ? FFN_CALL(__nv_bfloat16, 8) : FFN_CALL(__nv_bfloat16, 1);
  return v16 ? FFN_CALL(__half, 8) : FFN_CALL(__half, 1);
#undef FFN_CALL
}

}  // extern "C"
