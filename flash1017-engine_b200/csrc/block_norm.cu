// block_norm.cu -- the norms after one block and before the next, with the
// block's gate and the scaled residual add between them, in one pass over the
// rows; and its gradient.  The layer's own input norm (flash1017.rs:4880-4891)
// is the special case without a block output.
//
//   rms(v) = v / sqrt(mean(v^2) + eps)
//   b  = rms(y) * post_w   (y itself when post_w is NULL)
//   h  = alpha * residual + beta * gate * b       gate: none, [cols] or [rows]
//   xn = rms(h) * pre_w                           (optional; optional int8 codes)
//
// Backward, from the stored y and h, with dh the gradient that reaches h past
// the norm and dxn that of xn; u = dxn pre_w, r_v = 1 / sqrt(mean(v^2) + eps):
//   g        = dh + r_h (u - h r_h^2 mean(u h))
//   dres     = alpha g          dpre_w = sum_rows dxn h r_h
//   dgate    = beta sum g b     (over rows, or over columns)
//   v        = beta gate g post_w,  dpost_w = sum_rows beta gate g y r_y
//   dy       = r_y (v - y r_y^2 mean(v y))
//
// Rows stay in registers between the reductions: forward reads y and the
// residual once and writes h and xn once, backward reads four rows and writes
// two, so both are bound by DRAM.  Sums are f32 in a fixed order, without
// atomics.
#include <algorithm>

#include "ffn_internal.h"
#include "rowops.cuh"

namespace ffn {
namespace bn {

constexpr int kMaxCols = 16384;

__device__ __forceinline__ void stage16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
// Sum over the CTA's threads; s: 32 floats that no warp reads any more.
__device__ __forceinline__ float cta_sum(float v, float *s, int lane, int warp, int nw) {
  v = warp_sum(v);
  if (lane == 0) s[warp] = v;
  __syncthreads();
  return warp_sum(lane < nw ? s[lane] : 0.f);
}

struct FwdArgs {
  const void *y, *res;
  size_t ld_y, ld_r, ld_h, ld_x, ld_c;
  const float *post_w, *gate, *pre_w;
  int gate_kind;
  float alpha, beta, eps;
  void *h, *xn;
  int8_t *codes;
  float *code_scale;
  int rows;
  uint32_t cols, n_vec;
};

// Persistent, a row per CTA at a time; thread l holds the columns of pieces l,
// l + L, ... (8 or 16).  The parameters stay in its registers (P = beta gate_c
// post_w, pre_w); cp.async brings the CTA's next two rows into shared memory,
// every thread its own pieces (STAGED).  A CTA a row that loaded, reduced and
// re-read the parameters took 61 us for 8192 x 4096 bf16 (4.4 TB/s).
constexpr int kFwdStages = 3;
template <typename T, int VEC, int NV, int MT, bool STAGED>
__global__ void __launch_bounds__(MT, MT == 256 ? 3 : MT == 384 ? 2 : 1) fwd_kernel(const FwdArgs a) {
  __shared__ float s_red[2][3][32];
  extern __shared__ __align__(16) uint8_t s_dyn[];  // stages [kFwdStages][2 rows][NV][threads] of 16 bytes
  pdl_enter();
  const uint32_t l = threadIdx.x, L = blockDim.x;
  const int lane = l & 31, warp = l >> 5, nw = L >> 5;
  const T *src[2] = {(const T *)a.y, (const T *)a.res};
  const size_t ld[2] = {a.ld_y, a.ld_r};
  uint4 *st = reinterpret_cast<uint4 *>(s_dyn) + l;
  auto fetch = [&](int stage, long long row) {
    if (row < a.rows) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (src[w]) {
          const T *p = src[w] + (size_t)row * ld[w];
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (l + i * L < a.n_vec) stage16(st + ((stage * 2 + w) * NV + i) * L, p + (l + i * L) * VEC);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (STAGED) {
    for (int q = 0; q < kFwdStages - 1; ++q) fetch(q, blockIdx.x + (long long)q * gridDim.x);
    // pieces that no copy fills (past the row, absent rows) read as 0
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (!src[w] || l + i * L >= a.n_vec)
          for (int q = 0; q < kFwdStages; ++q) st[((q * 2 + w) * NV + i) * L] = make_uint4(0, 0, 0, 0);
  }
  float P[NV][VEC], pre[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
#pragma unroll
    for (int j = 0; j < VEC; ++j) P[i][j] = pre[i][j] = 0.f;
    if (v < a.n_vec) {
      if (a.pre_w) load_param<VEC>(a.pre_w, v, pre[i]);
      float w[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) P[i][j] = a.beta;
      if (a.post_w) {
        load_param<VEC>(a.post_w, v, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) P[i][j] *= w[j];
      }
      if (a.gate_kind == FFN_B200_GATE_CHANNEL) {
        load_param<VEC>(a.gate, v, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) P[i][j] *= w[j];
      }
    }
  }
  const float inv_n = 1.f / (float)a.cols;
  float gate = a.gate_kind == FFN_B200_GATE_TOKEN ? a.gate[blockIdx.x] : 1.f;  // the next row's
  int par = 0, stage = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1) {
    Raw<T, VEC> r[2][NV] = {};
    if constexpr (STAGED) {
      const int ahead = stage == 0 ? kFwdStages - 1 : stage - 1;  // two rows on: the stage read last
      fetch(ahead, row + (long long)(kFwdStages - 1) * gridDim.x);
      asm volatile("cp.async.wait_group %0;" ::"n"(kFwdStages - 1) : "memory");
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < NV; ++i) r[w][i] = *reinterpret_cast<const Raw<T, VEC> *>(st + ((stage * 2 + w) * NV + i) * L);
      stage = stage == kFwdStages - 1 ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (src[w])
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (l + i * L < a.n_vec) r[w][i] = load_raw<T, VEC>(src[w] + (size_t)row * ld[w], l + i * L);
    }
    float k = gate;
    if (a.gate_kind == FFN_B200_GATE_TOKEN && row + gridDim.x < a.rows) gate = a.gate[row + gridDim.x];
    if (a.post_w) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[VEC];
        unpack<T, VEC>(r[0][i], e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s = fmaf(e[j], e[j], s);
      }
      s = cta_sum(s, s_red[par][0], lane, warp, nw);
      k *= rsqrtf(fmaf(s, inv_n, a.eps));
    }
    float h[NV][VEC], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float y[VEC], e[VEC];
      unpack<T, VEC>(r[0][i], y);
      unpack<T, VEC>(r[1][i], e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        h[i][j] = fmaf(a.alpha, e[j], y[j] * k * P[i][j]);
        ss = fmaf(h[i][j], h[i][j], ss);
      }
      if (a.h && l + i * L < a.n_vec) store_vec<T, VEC>((T *)a.h + (size_t)row * a.ld_h, l + i * L, h[i]);
    }
    if (!a.pre_w) continue;
    ss = cta_sum(ss, s_red[par][1], lane, warp, nw);
    const float rh = rsqrtf(fmaf(ss, inv_n, a.eps));
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) h[i][j] = h[i][j] * rh * pre[i][j];
      if (l + i * L < a.n_vec) {
        if (a.xn) store_vec<T, VEC>((T *)a.xn + (size_t)row * a.ld_x, l + i * L, h[i]);
        if (a.codes)
#pragma unroll
          for (int j = 0; j < VEC; ++j) m = max(m, __float_as_uint(h[i][j]) & 0x7fffffffu);
      }
    }
    if (!a.codes) continue;
    // int8 codes of the f32 values (before xn's rounding), as quantize_int8
    uint32_t *sm = reinterpret_cast<uint32_t *>(s_red[par][2]);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) sm[warp] = m;
    __syncthreads();
    const Int8Row sc(__uint_as_float(__reduce_max_sync(0xffffffffu, lane < nw ? sm[lane] : 0u)));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (l + i * L < a.n_vec) store_codes<VEC>(a.codes + (size_t)row * a.ld_c + (size_t)(l + i * L) * VEC, h[i], sc);
    if (l == 0) a.code_scale[row] = sc.scale();
  }
}

struct BwdArgs {
  const void *src[4];               // y, h, dh, dxn; NULL: zeros
  size_t ld[4], ld_dr, ld_dy;
  const float *post_w, *gate, *pre_w;
  int gate_kind;
  float alpha, beta, eps;
  void *dres, *dy;
  float *dgate_tok;                 // [rows] or NULL
  float *part_pre, *part_br;        // [parts][cols] each, or NULL
  int rows;
  uint32_t cols, n_vec;
};

// Persistent, a row per CTA at a time; thread l holds the columns of pieces l,
// l + L, ...  What is the same for every row stays in its registers: pre_w,
// P = beta gate_c post_w (gate_c the per-channel gate, or 1), and two column
// sums, which it leaves in the workspace at the end (one partial row a CTA):
//   sum_rows dxn h r_h = dpre_w,  S = sum_rows beta gate_t g y r_y  (gate_t the
//   token's gate, or 1);  dpost_w = gate_c S,  dgate_c = post_w S
// The branch needs one more row sum, q = sum P g y: mean(v y) = gate_t q / cols,
// and a token's dgate is r_y q.
//
// STAGED: while a row is worked on, cp.async brings the CTA's next row into
// shared memory, every thread its own pieces, so a thread waits for its own
// copies alone.  Without that DRAM idled through both reductions, and with the
// parameters and three sums re-read per row the instructions took longer than
// the bytes (4093 x 5120 f32: 108 us unstaged, 100 us like this; 8192 x 4096
// bf16: 112 and 88 us).
template <typename T, int VEC, int NV, int MT, bool STAGED>
__global__ void __launch_bounds__(MT) bwd_kernel(const BwdArgs a) {
  __shared__ float4 s_red[2][32];
  __shared__ float s_q[2][32];
  extern __shared__ __align__(16) uint8_t s_dyn[];  // stages [2][4 rows][NV][threads] of 16 bytes
  pdl_enter();
  const uint32_t l = threadIdx.x, L = blockDim.x;
  const int lane = l & 31, warp = l >> 5, nw = L >> 5;
  float pre[NV][VEC], P[NV][VEC], c_pre[NV][VEC], c_br[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
#pragma unroll
    for (int j = 0; j < VEC; ++j) pre[i][j] = P[i][j] = c_pre[i][j] = c_br[i][j] = 0.f;
    if (v < a.n_vec) {
      if (a.src[3]) load_param<VEC>(a.pre_w, v, pre[i]);
      if (a.src[0]) {
        float w[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) P[i][j] = a.beta;
        if (a.post_w) {
          load_param<VEC>(a.post_w, v, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) P[i][j] *= w[j];
        }
        if (a.gate_kind == FFN_B200_GATE_CHANNEL) {
          load_param<VEC>(a.gate, v, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) P[i][j] *= w[j];
        }
      }
    }
  }
  const float inv_n = 1.f / (float)a.cols;
  uint4 *st = reinterpret_cast<uint4 *>(s_dyn) + l;
  auto fetch = [&](int stage, long long row) {
    if (row < a.rows) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (a.src[w]) {
          const T *p = (const T *)a.src[w] + (size_t)row * a.ld[w];
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (l + i * L < a.n_vec) stage16(st + ((stage * 4 + w) * NV + i) * L, p + (l + i * L) * VEC);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (STAGED) {  // pieces that no copy fills (past the row, absent rows) read as 0
    for (int q = 0; q < 8 * NV; ++q) st[q * L] = make_uint4(0, 0, 0, 0);
    fetch(0, blockIdx.x);
  }
  int par = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1) {
    // y, h, dh, dxn: in shared memory, read again in every phase (a piece is one
    // load), or in registers
    Raw<T, VEC> r[STAGED ? 1 : 4][STAGED ? 1 : NV] = {};
    auto piece = [&](int w, int i) {
      if constexpr (STAGED) return *reinterpret_cast<const Raw<T, VEC> *>(st + ((par * 4 + w) * NV + i) * L);
      else return r[w][i];
    };
    if constexpr (STAGED) {
      fetch(par ^ 1, row + gridDim.x);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (a.src[w])
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (l + i * L < a.n_vec) r[w][i] = load_raw<T, VEC>((const T *)a.src[w] + (size_t)row * a.ld[w], l + i * L);
    }
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);  // sum y^2, sum h^2, sum u h
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float y[VEC], h[VEC], d[VEC];
      unpack<T, VEC>(piece(0, i), y), unpack<T, VEC>(piece(1, i), h), unpack<T, VEC>(piece(3, i), d);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s.x = fmaf(y[j], y[j], s.x);
        s.y = fmaf(h[j], h[j], s.y);
        s.z = fmaf(d[j] * pre[i][j], h[j], s.z);
      }
    }
    s.x = warp_sum(s.x), s.y = warp_sum(s.y), s.z = warp_sum(s.z);
    if (lane == 0) s_red[par][warp] = s;
    __syncthreads();
    s = lane < nw ? s_red[par][lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    s.x = warp_sum(s.x), s.y = warp_sum(s.y), s.z = warp_sum(s.z);
    const float r_y = a.post_w ? rsqrtf(fmaf(s.x, inv_n, a.eps)) : 1.f;
    const float r_h = a.src[3] ? rsqrtf(fmaf(s.y, inv_n, a.eps)) : 0.f;
    const float m_h = s.z * inv_n * r_h * r_h;
    const float gt = a.gate_kind == FFN_B200_GATE_TOKEN && a.src[0] ? a.gate[row] : 1.f;
    const float k_br = a.beta * gt * r_y;
    float v[NV][VEC], q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float y[VEC], h[VEC], g[VEC], d[VEC];
      unpack<T, VEC>(piece(0, i), y), unpack<T, VEC>(piece(1, i), h), unpack<T, VEC>(piece(2, i), g), unpack<T, VEC>(piece(3, i), d);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        g[j] = fmaf(r_h, fmaf(d[j], pre[i][j], -h[j] * m_h), g[j]);
        c_pre[i][j] = fmaf(d[j], h[j] * r_h, c_pre[i][j]);
        c_br[i][j] = fmaf(g[j] * y[j], k_br, c_br[i][j]);
        v[i][j] = g[j] * P[i][j];
        q = fmaf(v[i][j], y[j], q);
        g[j] *= a.alpha;
      }
      if (a.dres && l + i * L < a.n_vec) store_vec<T, VEC>((T *)a.dres + (size_t)row * a.ld_dr, l + i * L, g);
    }
    if (!a.src[0]) continue;
    q = warp_sum(q);
    if (lane == 0) s_q[par][warp] = q;
    __syncthreads();
    q = warp_sum(lane < nw ? s_q[par][lane] : 0.f);
    if (a.dgate_tok && l == 0) a.dgate_tok[row] = r_y * q;
    if (a.dy) {
      const float m_y = a.post_w ? q * inv_n * r_y * r_y : 0.f, k = r_y * gt;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float y[VEC];
        unpack<T, VEC>(piece(0, i), y);
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = k * fmaf(-y[j], m_y, v[i][j]);
        if (l + i * L < a.n_vec) store_vec<T, VEC>((T *)a.dy + (size_t)row * a.ld_dy, l + i * L, y);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (l + i * L >= a.n_vec) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const size_t at = (size_t)blockIdx.x * a.cols + (size_t)(l + i * L) * VEC + j;
      if (a.part_pre) a.part_pre[at] = c_pre[i][j];
      if (a.part_br) a.part_br[at] = c_br[i][j];
    }
  }
}

// Column sums of the partial rows, 32 columns a CTA: warp w adds every 32nd row
// in order, then the 32 sums are added as a tree.  A few rows a warp, so all
// loads of a CTA are on their way at once.  Plane 0: dpre_w; plane 1: S, which
// gives dpost_w and a per-channel dgate.
struct ColArgs {
  const float *part[2];
  float *dpre, *dpost, *dgate;
  const float *post_w, *gate_c;
  int parts;
  uint32_t cols;
};
__global__ void __launch_bounds__(1024) colsum_kernel(const ColArgs a) {
  __shared__ float s[32][33];
  pdl_enter();
  const float *p = a.part[blockIdx.y];
  if (!p) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < a.cols) {
#pragma unroll 8
    for (int r = warp; r < a.parts; r += 32) sum += p[(size_t)r * a.cols + c];
  }
  s[warp][lane] = sum;
  __syncthreads();
  sum = warp_sum(s[lane][warp]);  // lane = partial, warp = column
  const uint32_t col = blockIdx.x * 32 + warp;
  if (lane || col >= a.cols) return;
  if (blockIdx.y == 0) a.dpre[col] = sum;
  else {
    if (a.dpost) a.dpost[col] = a.gate_c ? a.gate_c[col] * sum : sum;
    if (a.dgate) a.dgate[col] = a.post_w ? a.post_w[col] * sum : sum;
  }
}

// ------------------------------------------------------------------ launch
// Forward: 8 columns a thread up to 1024 columns, else 16: a row's reductions
// and addresses cost a thread about as many instructions as 8 columns do (8192 x
// 4096 bf16: 60 us with 8, 46 us with 16).
template <typename T, int VEC, int NV, int MT>
int launch_fwd_as(FwdArgs &a, cudaStream_t st) {
  constexpr bool STAGED = VEC > 1 && (size_t)kFwdStages * 2 * NV * MT * 16 <= 224 * 1024;
  const int threads = (int)((a.n_vec + 32 * NV - 1) / (32 * NV) * 32);
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(FFN_B200_EUNSUP, "block_norm: device index >= 64");
  const size_t smem = STAGED ? (size_t)kFwdStages * 2 * NV * threads * 16 : 0;
  static bool attr[64] = {false};
  if (STAGED && !attr[dev]) {
    FFN_CUDA_TRY(cudaFuncSetAttribute(fwd_kernel<T, VEC, NV, MT, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kFwdStages * 2 * NV * MT * 16));
    attr[dev] = true;
  }
  // as many CTAs as are resident at once: one more, and a second wave of whole
  // shares of the rows would follow (8192 x 4096 bf16: 51 us with half a wave more)
  static int resident[64][MT / 32 + 1] = {{0}};
  int &per_sm = resident[dev][threads / 32];
  if (per_sm == 0) {
    int n = 0;
    FFN_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fwd_kernel<T, VEC, NV, MT, STAGED>, threads, smem));
    per_sm = std::max(1, n);
  }
  const int grid = (int)std::min<long long>(a.rows, (long long)sm_count_of(dev) * per_sm);
  FFN_LAUNCH_PDL(FFN_B200_K_NORM, st, "block_norm", (fwd_kernel<T, VEC, NV, MT, STAGED>), grid, threads, smem, a);
  return 0;
}
template <typename T, int VEC>
int launch_fwd(FwdArgs &a, cudaStream_t st) {
  a.n_vec = a.cols / VEC;
  if (a.cols <= 1024) return launch_fwd_as<T, VEC, 8 / VEC, 128>(a, st);
  if (a.cols <= 4096) return launch_fwd_as<T, VEC, 16 / VEC, 256>(a, st);
  if (a.cols <= 6144) return launch_fwd_as<T, VEC, 16 / VEC, 384>(a, st);
  if (a.cols <= 8192) return launch_fwd_as<T, VEC, 16 / VEC, 512>(a, st);
  return launch_fwd_as<T, VEC, 16 / VEC, 1024>(a, st);
}

// Backward: 8 columns a thread (about 90 registers) up to 5120 columns for f32,
// where the staged rows leave room for one CTA an SM anyway, and for single
// elements, and up to 1024 for 16-bit types; else 16, which halves the reductions'
// share of the instructions.  Above 8192 columns that is a CTA of up to 1024 threads
// with 64 registers each, which spills (bf16 628 bytes stored and 672 loaded a
// thread, single elements 1246 and 1128) and has no stages: 2048 x 16384 bf16 takes
// 217 us, where its bytes would take 62.
constexpr int kStageMax = 224 * 1024;
struct BwdShape {
  int per, threads;  // columns a thread, threads
};
BwdShape bwd_shape(uint32_t cols, int vec) {
  const int per = cols <= (vec == 8 ? 1024u : 5120u) ? 8 : 16;
  return {per, (int)((cols + per * 32 - 1) / (per * 32) * 32)};
}
int bwd_parts(size_t rows, uint32_t cols, int vec, int sms) {  // CTAs: as many as stay resident
  const BwdShape s = bwd_shape(cols, vec);
  return (int)std::min<size_t>(rows, (size_t)sms * std::min(8, std::max(1, (s.per == 8 ? 640 : 512) / s.threads)));
}

template <typename T, int VEC, int NV, int MT, bool STAGED>
int launch_bwd_as(BwdArgs &a, int parts, int threads, cudaStream_t st) {
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(FFN_B200_EUNSUP, "block_norm_bwd: device index >= 64");
  static bool attr[64] = {false};
  if (STAGED && !attr[dev]) {
    FFN_CUDA_TRY(cudaFuncSetAttribute(bwd_kernel<T, VEC, NV, MT, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStageMax));
    attr[dev] = true;
  }
  const size_t smem = STAGED ? (size_t)8 * NV * threads * 16 : 0;
  FFN_LAUNCH_PDL(FFN_B200_K_NORM, st, "block_norm_bwd", (bwd_kernel<T, VEC, NV, MT, STAGED>), parts, threads, smem, a);
  return 0;
}
template <typename T, int VEC>
int launch_bwd(BwdArgs &a, int parts, cudaStream_t st) {
  a.n_vec = a.cols / VEC;
  const BwdShape s = bwd_shape(a.cols, VEC);
  constexpr int N8 = 8 / VEC, N16 = 16 / VEC;
  if (s.per == 8) return launch_bwd_as<T, VEC, N8, 640, (VEC > 1)>(a, parts, s.threads, st);
  if (s.threads > 512) return launch_bwd_as<T, VEC, N16, 1024, false>(a, parts, s.threads, st);
  if (VEC > 1 && (size_t)8 * N16 * s.threads * 16 <= (size_t)kStageMax)
    return launch_bwd_as<T, VEC, N16, 512, (VEC > 1)>(a, parts, s.threads, st);
  return launch_bwd_as<T, VEC, N16, 512, false>(a, parts, s.threads, st);
}

int check_desc(const char *what, const ffn_b200_block_norm_desc *d) {
  const std::string w(what);
  if (!d) return fail(FFN_B200_EINVAL, w + ": null descriptor");
  if (!dtype_ok(d->dtype)) return fail(FFN_B200_EINVAL, w + ": unknown dtype");
  if (d->cols == 0 || d->cols > (size_t)kMaxCols) return fail(FFN_B200_EUNSUP, w + ": cols must be in 1..16384");
  if (d->rows > 0x7fffffffu) return fail(FFN_B200_EINVAL, w + ": too many rows");
  if (d->gate_kind != FFN_B200_GATE_NONE && d->gate_kind != FFN_B200_GATE_CHANNEL && d->gate_kind != FFN_B200_GATE_TOKEN)
    return fail(FFN_B200_EINVAL, w + ": unknown gate_kind");
  const bool no_gates = d->rows == 0 && d->gate_kind == FFN_B200_GATE_TOKEN;  // an empty array's address is null
  if (!no_gates && (d->gate_kind != FFN_B200_GATE_NONE) != (d->gate != nullptr))
    return fail(FFN_B200_EINVAL, w + ": gate and gate_kind go together");
  if (!(d->eps >= 0.f)) return fail(FFN_B200_EINVAL, w + ": eps must not be negative");
  if (((uintptr_t)d->post_w | (uintptr_t)d->pre_w | (uintptr_t)d->gate) % 4)
    return fail(FFN_B200_EINVAL, w + ": parameters must be 4-byte aligned");
  return 0;
}
bool params16(const ffn_b200_block_norm_desc *d) {
  return (((uintptr_t)d->post_w | (uintptr_t)d->pre_w |
           (d->gate_kind == FFN_B200_GATE_CHANNEL ? (uintptr_t)d->gate : 0)) & 15) == 0;
}

}  // namespace bn
}  // namespace ffn

using namespace ffn;

extern "C" {

int ffn_b200_block_norm(const ffn_b200_block_norm_desc *d, const void *y, size_t ld_y, const void *residual, size_t ld_res,
                        void *h, size_t ld_h, void *xn, size_t ld_xn, int8_t *codes, size_t ld_codes, float *code_scales,
                        void *stream) {
  using namespace ffn::bn;
  if (int rc = check_desc("block_norm", d)) return rc;
  if (d->rows == 0) return 0;
  if (!y && !residual) return fail(FFN_B200_EINVAL, "block_norm: neither y nor residual");
  if (!h && !xn && !codes) return fail(FFN_B200_EINVAL, "block_norm: no output");
  if ((xn || codes) && !d->pre_w) return fail(FFN_B200_EINVAL, "block_norm: xn and codes need pre_w");
  if (!y && (d->post_w || d->gate)) return fail(FFN_B200_EINVAL, "block_norm: post_w and gate need y");
  if ((codes == nullptr) != (code_scales == nullptr))
    return fail(FFN_B200_EINVAL, "block_norm: codes and code_scales go together");
  if (d->rows > 1 && ((y && ld_y < d->cols) || (residual && ld_res < d->cols) || (h && ld_h < d->cols) ||
                      (xn && ld_xn < d->cols) || (codes && ld_codes < d->cols)))
    return fail(FFN_B200_EINVAL, "block_norm: rows overlap");
  const size_t es = dtype_bytes(d->dtype);
  if (((uintptr_t)y | (uintptr_t)residual | (uintptr_t)h | (uintptr_t)xn) % es)
    return fail(FFN_B200_EINVAL, "block_norm: rows must be aligned to their type");
  if ((uintptr_t)code_scales % 4) return fail(FFN_B200_EINVAL, "block_norm: code_scales must be 4-byte aligned");
  FwdArgs a{};
  a.y = y, a.res = residual, a.h = h, a.xn = xn, a.codes = codes, a.code_scale = code_scales;
  a.ld_y = ld_y, a.ld_r = ld_res, a.ld_h = ld_h, a.ld_x = ld_xn, a.ld_c = ld_codes;
  a.post_w = d->post_w, a.gate = d->gate, a.pre_w = xn || codes ? d->pre_w : nullptr;
  a.gate_kind = d->gate_kind;
  a.alpha = d->alpha, a.beta = d->beta, a.eps = d->eps;
  a.rows = (int)d->rows;
  a.cols = (uint32_t)d->cols;
  const bool v16 = d->cols * es % 16 == 0 && rows16(y, ld_y, es) && rows16(residual, ld_res, es) && rows16(h, ld_h, es) &&
                   rows16(xn, ld_xn, es) && params16(d) && (!codes || (((uintptr_t)codes | ld_codes) & 7) == 0);
  cudaStream_t st = (cudaStream_t)stream;
  if (d->dtype == FFN_B200_DT_F32) return v16 ? launch_fwd<float, 4>(a, st) : launch_fwd<float, 1>(a, st);
  if (d->dtype == FFN_B200_DT_BF16) return v16 ? launch_fwd<__nv_bfloat16, 8>(a, st) : launch_fwd<__nv_bfloat16, 1>(a, st);
  return v16 ? launch_fwd<__half, 8>(a, st) : launch_fwd<__half, 1>(a, st);
}

size_t ffn_b200_block_norm_bwd_ws_bytes(const ffn_b200_block_norm_desc *d) {
  using namespace ffn::bn;
  if (!d || d->cols == 0 || d->cols > (size_t)kMaxCols || !dtype_ok(d->dtype)) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    dev = -1;
  }
  // whatever the pointers' alignment will allow
  const int sms = sm_count_of(dev), vec = (int)(16 / dtype_bytes(d->dtype));
  const int parts = std::max(bwd_parts(d->rows, (uint32_t)d->cols, vec, sms), bwd_parts(d->rows, (uint32_t)d->cols, 1, sms));
  return (size_t)parts * d->cols * 2 * sizeof(float) + 16;
}

int ffn_b200_block_norm_bwd(const ffn_b200_block_norm_desc *d, const void *y, size_t ld_y, const void *h, size_t ld_h,
                            const void *dh, size_t ld_dh, const void *dxn, size_t ld_dxn, void *dresidual, size_t ld_dres,
                            void *dy, size_t ld_dy, float *dpost_w, float *dgate, float *dpre_w, void *ws, size_t ws_bytes,
                            void *stream) {
  using namespace ffn::bn;
  if (int rc = check_desc("block_norm_bwd", d)) return rc;
  if ((dpost_w && !d->post_w) || (dgate && d->gate_kind == FFN_B200_GATE_NONE))
    return fail(FFN_B200_EINVAL, "block_norm_bwd: a gradient of a parameter that is not there");
  if (((uintptr_t)dpost_w | (uintptr_t)dgate | (uintptr_t)dpre_w) % 4)
    return fail(FFN_B200_EINVAL, "block_norm_bwd: parameter gradients must be 4-byte aligned");
  const bool chan = d->gate_kind == FFN_B200_GATE_CHANNEL && dgate;
  cudaStream_t st = (cudaStream_t)stream;
  if (d->rows == 0) {  // sums over no rows
    if (dpre_w) FFN_CUDA_TRY(cudaMemsetAsync(dpre_w, 0, d->cols * sizeof(float), st));
    if (dpost_w) FFN_CUDA_TRY(cudaMemsetAsync(dpost_w, 0, d->cols * sizeof(float), st));
    if (chan) FFN_CUDA_TRY(cudaMemsetAsync(dgate, 0, d->cols * sizeof(float), st));
    return 0;
  }
  if (!dh && !dxn) return fail(FFN_B200_EINVAL, "block_norm_bwd: neither dh nor dxn");
  if (dxn && (!h || !d->pre_w)) return fail(FFN_B200_EINVAL, "block_norm_bwd: dxn needs h and pre_w");
  if (dpre_w && !dxn) return fail(FFN_B200_EINVAL, "block_norm_bwd: dpre_w needs dxn");
  if ((dy || dpost_w || dgate) && !y && d->rows) return fail(FFN_B200_EINVAL, "block_norm_bwd: dy, dpost_w and dgate need y");
  if (d->rows > 1 && ((y && ld_y < d->cols) || (h && dxn && ld_h < d->cols) || (dh && ld_dh < d->cols) ||
                      (dxn && ld_dxn < d->cols) || (dresidual && ld_dres < d->cols) || (dy && ld_dy < d->cols)))
    return fail(FFN_B200_EINVAL, "block_norm_bwd: rows overlap");
  const size_t es = dtype_bytes(d->dtype);
  if (((uintptr_t)y | (uintptr_t)h | (uintptr_t)dh | (uintptr_t)dxn | (uintptr_t)dresidual | (uintptr_t)dy) % es)
    return fail(FFN_B200_EINVAL, "block_norm_bwd: rows must be aligned to their type");
  BwdArgs a{};
  const bool branch = dy || dpost_w || dgate;
  a.src[0] = branch ? y : nullptr, a.src[1] = dxn ? h : nullptr, a.src[2] = dh, a.src[3] = dxn;
  a.ld[0] = ld_y, a.ld[1] = ld_h, a.ld[2] = ld_dh, a.ld[3] = ld_dxn, a.ld_dr = ld_dres, a.ld_dy = ld_dy;
  a.post_w = branch ? d->post_w : nullptr, a.gate = d->gate, a.pre_w = d->pre_w;
  a.gate_kind = d->gate_kind;
  a.alpha = d->alpha, a.beta = d->beta, a.eps = d->eps;
  a.dres = dresidual, a.dy = dy;
  a.dgate_tok = d->gate_kind == FFN_B200_GATE_TOKEN ? dgate : nullptr;
  a.rows = (int)d->rows;
  a.cols = (uint32_t)d->cols;
  bool v16 = d->cols * es % 16 == 0 && rows16(dresidual, ld_dres, es) && rows16(dy, ld_dy, es) && params16(d);
  for (int i = 0; i < 4; ++i) v16 = v16 && rows16(a.src[i], a.ld[i], es);
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  const int parts = bwd_parts(d->rows, a.cols, v16 ? (int)(16 / es) : 1, sm_count_of(dev));
  const bool any = dpre_w || dpost_w || chan;
  if (any) {
    if (!ws || (uintptr_t)ws % 4) return fail(FFN_B200_EINVAL, "block_norm_bwd: the workspace is null or misaligned");
    if (ws_bytes < ffn_b200_block_norm_bwd_ws_bytes(d)) return fail(FFN_B200_ENOSPC, "block_norm_bwd: workspace too small");
  }
  if (dpre_w) a.part_pre = (float *)ws;
  if (dpost_w || chan) a.part_br = (float *)ws + (size_t)parts * d->cols;
  int rc;
  if (d->dtype == FFN_B200_DT_F32) rc = v16 ? launch_bwd<float, 4>(a, parts, st) : launch_bwd<float, 1>(a, parts, st);
  else if (d->dtype == FFN_B200_DT_BF16) rc = v16 ? launch_bwd<__nv_bfloat16, 8>(a, parts, st) : launch_bwd<__nv_bfloat16, 1>(a, parts, st);
  else rc = v16 ? launch_bwd<__half, 8>(a, parts, st) : launch_bwd<__half, 1>(a, parts, st);
  if (rc || !any) return rc;
  ColArgs c{};
  c.part[0] = a.part_pre, c.part[1] = a.part_br;
  c.dpre = dpre_w, c.dpost = dpost_w, c.dgate = chan ? dgate : nullptr;
  c.post_w = d->post_w, c.gate_c = d->gate_kind == FFN_B200_GATE_CHANNEL ? d->gate : nullptr;
  c.parts = parts;
  c.cols = a.cols;
  FFN_LAUNCH_PDL(FFN_B200_K_NORM, st, "colsum_kernel", colsum_kernel, dim3((a.cols + 31) / 32, 2), 1024, 0, c);
  return 0;
}

}  // extern "C"
