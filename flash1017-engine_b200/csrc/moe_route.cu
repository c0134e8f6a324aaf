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
// contiguous segment of the pairs.  A warp ranks 32 pairs at a time with
// match.any (lanes of the same expert, in lane order), so the order inside an
// expert is the pair order.  Counts per (segment, expert) sit in shared
// memory; the CTAs of the cluster read each other's totals over distributed
// shared memory, which saves the second and third launch and the workspace
// that a grid-wide sort would need.  Bound by latency, not by bytes: 8 bytes
// a pair.
constexpr int kSortThreads = 1024;
constexpr int kSortCluster = 8;
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
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(b) : "memory");
  return v;
}

__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const SortArgs a) {
  extern __shared__ int s_cnt[];  // [segs][n_local], then [n_local] totals, then [n_local + 1] offsets
  __shared__ int s_warp[32];
  __shared__ int s_carry;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), nrank = cluster_size();
  int *tot = s_cnt + a.segs * a.n_local, *off = tot + a.n_local;
  for (int i = tid; i < a.segs * a.n_local; i += kSortThreads) s_cnt[i] = 0;
  __syncthreads();

  // pass 1: counts per segment
  const long long s0 = ((long long)rank * a.segs + warp) * a.per_seg;
  const int p0 = (int)min(s0, (long long)a.n_pairs), p1 = (int)min(s0 + a.per_seg, (long long)a.n_pairs);
  int *mine = s_cnt + warp * a.n_local;
  if (warp < a.segs) {
    for (int p = p0; p < p1; p += 32) {
      int e = -1;
      if (p + lane < p1) {
        // unsigned: ids below e_begin, and the top-k step's "no candidate"
        // 0x7fffffff, fall outside like those at or above the range's end
        const uint32_t r = (uint32_t)__ldg(a.idx + p + lane) - (uint32_t)a.e_begin;
        if (r < (uint32_t)a.n_local) e = (int)r;
      }
      const uint32_t same = __match_any_sync(0xffffffffu, e);
      if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  // counts -> exclusive prefix over this CTA's segments; totals
  for (int e = tid; e < a.n_local; e += kSortThreads) {
    int run = 0;
    for (int s = 0; s < a.segs; ++s) {
      const int c = s_cnt[s * a.n_local + e];
      s_cnt[s * a.n_local + e] = run;
      run += c;
    }
    tot[e] = run;
  }
  __syncthreads();  // the cluster barrier is .aligned: whole warps arrive
  cluster_arrive();
  cluster_wait();
  // exclusive prefix over the experts of the cluster's totals; the pairs of
  // lower-ranked CTAs come first inside an expert
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int e0 = 0; e0 < a.n_local; e0 += kSortThreads) {
    const int e = e0 + tid;
    int all = 0, before = 0;
    if (e < a.n_local)
      for (uint32_t r = 0; r < nrank; ++r) {
        const int c = r == rank ? tot[e] : peer_int(tot + e, r);
        all += c;
        if (r < rank) before += c;
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
    if (e < a.n_local) {
      off[e] = first + before;
      if (rank == 0) a.offsets[e] = first;
    }
    __syncthreads();
    if (tid == 0) s_carry += s_warp[31];
    __syncthreads();
  }
  const int total = s_carry;
  if (rank == 0 && tid == 0) a.offsets[a.n_local] = total;
  cluster_arrive();  // the reads of the peers' totals are done; waited for at the end

  // pass 2: rows
  if (warp < a.segs) {
    for (int p = p0; p < p1; p += 32) {
      int e = -1;
      if (p + lane < p1) {
        const uint32_t r = (uint32_t)__ldg(a.idx + p + lane) - (uint32_t)a.e_begin;
        if (r < (uint32_t)a.n_local) e = (int)r;
      }
      const uint32_t same = __match_any_sync(0xffffffffu, e);
      const int base = e >= 0 ? mine[e] : 0;
      __syncwarp();
      if (e >= 0 && lane == __ffs(same) - 1) mine[e] = base + __popc(same);
      __syncwarp();
      const int row = e >= 0 ? off[e] + base + __popc(same & ((1u << lane) - 1u)) : -1;
      if (p + lane < p1) {
        if (a.pos) a.pos[p + lane] = row;
        if (a.src && row >= 0) a.src[row] = p + lane;
      }
    }
  }
  if (a.src)  // rows behind the last local pair
    for (long long r = total + (long long)rank * kSortThreads + tid; r < a.n_pairs; r += (long long)nrank * kSortThreads)
      a.src[r] = -1;
  __syncwarp();
  cluster_wait();
}

// (row, piece) of flat item i; 32-bit division where the items allow it
__device__ __forceinline__ int split_item(long long i, uint32_t n_vec, bool small, uint32_t &v) {
  if (small) {
    const uint32_t t = (uint32_t)i / n_vec;
    v = (uint32_t)i - t * n_vec;
    return (int)t;
  }
  const long long t = i / n_vec;
  v = (uint32_t)(i - t * n_vec);
  return (int)t;
}

// ------------------------------------------------- permute (rows of bytes)
// Flat over (token, piece of BYTES): each piece is read once and written to
// the token's rows.  DRAM-bound by the written rows.
template <int BYTES>
__global__ void __launch_bounds__(256) permute_kernel(const uint8_t *x, size_t ld_x, const int32_t *pos, uint8_t *out,
                                                      size_t ld_out, int n_tok, int top_k, uint32_t n_vec,
                                                      uint32_t out_rows, const float *x_scale, float *out_scale) {
  using R = typename RawOf<BYTES>::type;
  pdl_enter();
  const long long total = (long long)n_tok * n_vec, step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    uint32_t v;
    const int t = split_item(i, n_vec, total <= 0xffffffffLL, v);
    const R r = reinterpret_cast<const R *>(x + (size_t)t * ld_x)[v];
    const float s = x_scale && v == 0 ? __ldg(x_scale + t) : 0.f;
    const int32_t *pp = pos + (size_t)t * top_k;
    for (int k = 0; k < top_k; ++k) {
      const uint32_t p = (uint32_t)__ldg(pp + k);
      if (p >= out_rows) continue;
      reinterpret_cast<R *>(out + (size_t)p * ld_out)[v] = r;
      if (x_scale && v == 0) out_scale[p] = s;
    }
  }
}

// ----------------------------------------------------------------- combine
// Flat over (token, piece of VEC elements); kAhead rows are loaded before the
// first is used.  DRAM-bound by the experts' rows.
constexpr int kAhead = 4;
template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_rows_kernel(const T *y, size_t ld_y, uint32_t y_rows, const int32_t *pos,
                                                           const float *w, const T *residual, size_t ld_r, T *out,
                                                           size_t ld_o, int n_tok, int top_k, uint32_t n_vec) {
  pdl_enter();
  const long long total = (long long)n_tok * n_vec, step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
    uint32_t v;
    const int t = split_item(i, n_vec, total <= 0xffffffffLL, v);
    const int32_t *pp = pos + (size_t)t * top_k;
    const float *ww = w ? w + (size_t)t * top_k : nullptr;
    Raw<T, VEC> rr = {};
    if (residual) rr = load_raw<T, VEC>(residual + (size_t)t * ld_r, v);
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    for (int k0 = 0; k0 < top_k; k0 += kAhead) {
      Raw<T, VEC> r[kAhead];
      float f[kAhead];
      bool on[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        on[q] = false;
        if (k0 + q < top_k) {
          const uint32_t p = (uint32_t)__ldg(pp + k0 + q);
          on[q] = p < y_rows;
          if (on[q]) {
            r[q] = load_raw<T, VEC>(y + (size_t)p * ld_y, v);
            f[q] = ww ? __ldg(ww + k0 + q) : 1.f;
          }
        }
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
        if (on[q]) {
          float e[VEC];
          unpack<T, VEC>(r[q], e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = fmaf(f[q], e[j], acc[j]);
        }
    }
    if (residual) {
      float e[VEC];
      unpack<T, VEC>(rr, e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += e[j];
    }
    store_vec<T, VEC>(out + (size_t)t * ld_o, v, acc);
  }
}

// ------------------------------------------------------- combine, backward
// TPT threads (one warp, or the CTA) a token: the token's gradient row is read
// once per kBack choices, each choice's row of y once, each row of dy written
// once; the kBack dot products are reduced together.
constexpr int kBack = 8;
template <typename T, int VEC, int TPT>
__global__ void __launch_bounds__(256) combine_bwd_kernel(const T *dout, size_t ld_d, const T *y, size_t ld_y,
                                                          uint32_t y_rows, const int32_t *pos, const float *w, T *dy,
                                                          size_t ld_dy, float *dw, int n_tok, int top_k, uint32_t n_vec) {
  constexpr int kTok = 256 / TPT;
  __shared__ float s_red[8][kBack];
  pdl_enter();
  const int lane = threadIdx.x % TPT, sub = threadIdx.x / TPT;
  for (long long t0 = (long long)blockIdx.x * kTok; t0 < n_tok; t0 += (long long)gridDim.x * kTok) {
    const long long t = t0 + sub;
    const bool live = t < n_tok;
    const int32_t *pp = pos + (size_t)(live ? t : 0) * top_k;
    const float *ww = w ? w + (size_t)(live ? t : 0) * top_k : nullptr;
    const T *drow = dout + (size_t)(live ? t : 0) * ld_d;
    for (int k0 = 0; k0 < top_k; k0 += kBack) {
      uint32_t p[kBack];
      float f[kBack], dot[kBack];
#pragma unroll
      for (int q = 0; q < kBack; ++q) {
        p[q] = live && k0 + q < top_k ? (uint32_t)__ldg(pp + k0 + q) : 0xffffffffu;
        if (p[q] >= y_rows) p[q] = 0xffffffffu;
        f[q] = ww && p[q] != 0xffffffffu ? __ldg(ww + k0 + q) : 1.f;
        dot[q] = 0.f;
      }
      for (uint32_t v = lane; live && v < n_vec; v += TPT) {
        float d[VEC];
        unpack<T, VEC>(load_raw<T, VEC>(drow, v), d);
        if (dw) {
          Raw<T, VEC> r[kBack];
#pragma unroll
          for (int q = 0; q < kBack; ++q)
            if (p[q] != 0xffffffffu) r[q] = load_raw<T, VEC>(y + (size_t)p[q] * ld_y, v);
#pragma unroll
          for (int q = 0; q < kBack; ++q)
            if (p[q] != 0xffffffffu) {
              float e[VEC];
              unpack<T, VEC>(r[q], e);
#pragma unroll
              for (int j = 0; j < VEC; ++j) dot[q] = fmaf(d[j], e[j], dot[q]);
            }
        }
        if (dy) {
#pragma unroll
          for (int q = 0; q < kBack; ++q)
            if (p[q] != 0xffffffffu) {
              float e[VEC];
#pragma unroll
              for (int j = 0; j < VEC; ++j) e[j] = f[q] * d[j];
              store_vec<T, VEC>(dy + (size_t)p[q] * ld_dy, v, e);
            }
        }
      }
      if (dw) {
#pragma unroll
        for (int q = 0; q < kBack; ++q) dot[q] = warp_sum(dot[q]);
        if (TPT > 32) {
          if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int q = 0; q < kBack; ++q) s_red[threadIdx.x >> 5][q] = dot[q];
          __syncthreads();
          if (threadIdx.x < kBack && live && k0 + (int)threadIdx.x < top_k) {
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < 8; ++g) s += s_red[g][threadIdx.x];
            dw[(size_t)t * top_k + k0 + threadIdx.x] = s;
          }
          __syncthreads();
        } else if (live) {
#pragma unroll
          for (int q = 0; q < kBack; ++q)
            if (lane == q && k0 + q < top_k) dw[(size_t)t * top_k + k0 + q] = dot[q];
        }
      }
    }
  }
}

// ------------------------------------------------------------------ launch
int flat_grid(long long items) {  // 256 items a CTA, four waves of 8 CTAs an SM at most
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  return (int)std::max(1LL, std::min<long long>((items + 255) / 256, (long long)sm_count_of(dev) * 32));
}

template <int BYTES>
int launch_permute(const void *x, size_t ld_x, const int32_t *pos, void *out, size_t ld_out, size_t n_tok, size_t top_k,
                   size_t row_bytes, size_t out_rows, const float *xs, float *os, cudaStream_t st) {
  const uint32_t n_vec = (uint32_t)(row_bytes / BYTES);
  FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "permute_kernel", (permute_kernel<BYTES>), flat_grid((long long)n_tok * n_vec), 256, 0,
                 (const uint8_t *)x, ld_x, pos, (uint8_t *)out, ld_out, (int)n_tok, (int)top_k, n_vec, (uint32_t)out_rows,
                 xs, os);
  return 0;
}

template <typename T, int VEC>
int launch_combine_rows(const void *y, size_t ld_y, size_t y_rows, const int32_t *pos, const float *w, const void *res,
                        size_t ld_r, void *out, size_t ld_o, size_t n_tok, size_t top_k, size_t cols, cudaStream_t st) {
  const uint32_t n_vec = (uint32_t)(cols / VEC);
  FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "combine_rows_kernel", (combine_rows_kernel<T, VEC>),
                 flat_grid((long long)n_tok * n_vec), 256, 0, (const T *)y, ld_y, (uint32_t)y_rows, pos, w, (const T *)res,
                 ld_r, (T *)out, ld_o, (int)n_tok, (int)top_k, n_vec);
  return 0;
}

template <typename T, int VEC>
int launch_combine_bwd(const void *dout, size_t ld_d, const void *y, size_t ld_y, size_t y_rows, const int32_t *pos,
                       const float *w, void *dy, size_t ld_dy, float *dw, size_t n_tok, size_t top_k, size_t cols,
                       cudaStream_t st) {
  const uint32_t n_vec = (uint32_t)(cols / VEC);
  // a warp a token up to 4 pieces a lane; a CTA a token above
  if (n_vec <= 128) {
    const int grid = flat_grid((long long)n_tok * 32);
    FFN_LAUNCH_PDL(FFN_B200_K_ROUTE, st, "combine_bwd_kernel", (combine_bwd_kernel<T, VEC, 32>), grid, 256, 0,
                   (const T *)dout, ld_d, (const T *)y, ld_y, (uint32_t)y_rows, pos, w, (T *)dy, ld_dy, dw, (int)n_tok,
                   (int)top_k, n_vec);
  } else {
    const int grid = flat_grid((long long)n_tok * 256);
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
  // One CTA up to 2048 pairs (two groups of 32 a warp): no cluster to gather.
  const int nclu = a.n_pairs <= 2048 ? 1 : kSortCluster;
  const int groups = (a.n_pairs + 31) / 32, per_cta = (groups + nclu - 1) / nclu;
  a.segs = std::max(1, std::min({kSortThreads / 32, kSortCounts / a.n_local, per_cta}));
  a.per_seg = std::max(1, (per_cta + a.segs - 1) / a.segs) * 32;
  const size_t smem = ((size_t)a.segs * a.n_local + 2 * (size_t)a.n_local) * sizeof(int);
  static bool attr[64] = {false};
  if (!attr[dev]) {
    FFN_CUDA_TRY(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (kSortCounts + 2 * 4096) * (int)sizeof(int)));
    attr[dev] = true;
  }
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
  if (n_tok == 0) return 0;
  if (!x || !pos || !out) return fail(FFN_B200_EINVAL, "moe_permute: null pointer");
  if ((x_scale == nullptr) != (out_scale == nullptr))
    return fail(FFN_B200_EINVAL, "moe_permute: x_scale and out_scale go together");
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
  const bool v16 = cols * es % 16 == 0 && rows16(dw ? y : nullptr, ld_y, es) && rows16(dout, ld_dout, es) && rows16(dy, ld_dy, es);
  cudaStream_t st = (cudaStream_t)stream;
#define FFN_CALL(T, V) launch_combine_bwd<T, V>(dout, ld_dout, y, ld_y, y_rows, pos, w, dy, ld_dy, dw, n_tok, top_k, cols, st)
  if (dtype == FFN_B200_DT_F32) return v16 ? FFN_CALL(float, 4) : FFN_CALL(float, 1);
  if (dtype == FFN_B200_DT_BF16) return v16 ? FFN_CALL(__nv_bfloat16, 8) : FFN_CALL(__nv_bfloat16, 1);
  return v16 ? FFN_CALL(__half, 8) : FFN_CALL(__half, 1);
#undef FFN_CALL
}

}  // extern "C"
