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

// Sum of NV per-thread values over the threads of a row: a warp, or the CTA
// (s: 32 x NV floats, alternated by the caller between consecutive calls).
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float *s) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (WARP) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[warp * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < nw ? s[lane * N + i] : 0.f);
}
template <bool WARP>
__device__ __forceinline__ float row_max(float v, float *s) {
  v = warp_max(v);
  if (WARP) return v;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) s[warp] = v;
  __syncthreads();
  return warp_max(lane < nw ? s[lane] : 0.f);
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

// A row per warp (short rows, 8 a CTA) or per CTA; thread l of the row holds
// pieces l, l + L, ... of VEC elements, NV at most.
template <typename T, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) fwd_kernel(const FwdArgs a) {
  __shared__ float s_red[3][32];
  pdl_enter();
  const uint32_t l = WARP ? threadIdx.x & 31 : threadIdx.x, L = WARP ? 32 : blockDim.x;
  const long long row = WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;  // whole warps; a CTA's rows are all in range otherwise
  float h[NV][VEC];
  const T *yr = (const T *)a.y + (size_t)row * a.ld_y, *rr = (const T *)a.res + (size_t)row * a.ld_r;
  Raw<T, VEC> ry[NV] = {}, rres[NV] = {};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
    if (v < a.n_vec) {
      if (a.y) ry[i] = load_raw<T, VEC>(yr, v);
      if (a.res) rres[i] = load_raw<T, VEC>(rr, v);
    }
  }
  float ry_inv = 1.f;
  if (a.y && a.post_w) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float e[VEC];
      unpack<T, VEC>(ry[i], e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] = fmaf(e[j], e[j], s[0]);
    }
    row_sum<WARP, 1>(s, s_red[0]);
    ry_inv = 1.f / sqrtf(s[0] / (float)a.cols + a.eps);
  }
  const float gt = a.gate_kind == FFN_B200_GATE_TOKEN ? __ldg(a.gate + row) : 1.f;
  float ss[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[i][j] = 0.f;
    if (v < a.n_vec) {
      if (a.y) {
        unpack<T, VEC>(ry[i], h[i]);
        if (a.post_w) {
          float w[VEC];
          load_param<VEC>(a.post_w, v, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] = h[i][j] * ry_inv * w[j];
        }
        if (a.gate_kind == FFN_B200_GATE_CHANNEL) {
          float w[VEC];
          load_param<VEC>(a.gate, v, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] *= a.beta * gt;
      }
      if (a.res) {
        float e[VEC];
        unpack<T, VEC>(rres[i], e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = fmaf(a.alpha, e[j], h[i][j]);
      }
      if (a.h) store_vec<T, VEC>((T *)a.h + (size_t)row * a.ld_h, v, h[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss[0] = fmaf(h[i][j], h[i][j], ss[0]);
    }
  }
  if (!a.pre_w) return;
  row_sum<WARP, 1>(ss, s_red[1]);
  const float rh = 1.f / sqrtf(ss[0] / (float)a.cols + a.eps);
  float amax = 0.f;
  bool fin = true;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
    if (v < a.n_vec) {
      float w[VEC];
      load_param<VEC>(a.pre_w, v, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        h[i][j] = h[i][j] * rh * w[j];
        amax = fmaxf(amax, fabsf(h[i][j]));
        fin = fin && isfinite(h[i][j]);
      }
      if (a.xn) store_vec<T, VEC>((T *)a.xn + (size_t)row * a.ld_x, v, h[i]);
    }
  }
  if (!a.codes) return;
  // int8 codes of the f32 values (before xn's rounding), as quantize_int8
  amax = row_max<WARP>(fin ? amax : INFINITY, s_red[2]);
  const float sc = int8_scale(amax);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
    if (v < a.n_vec) store_codes<VEC>(a.codes + (size_t)row * a.ld_c + (size_t)v * VEC, h[i], sc);
  }
  if (l == 0) a.code_scale[row] = sc;
}

struct BwdArgs {
  const void *y, *h, *dh, *dxn;
  size_t ld_y, ld_h, ld_dh, ld_dx, ld_dr, ld_dy;
  const float *post_w, *gate, *pre_w;
  int gate_kind;
  float alpha, beta, eps;
  void *dres, *dy;
  float *dgate_tok;                 // [rows] or NULL
  float *part_pre, *part_post, *part_gate;  // [parts][cols] each, or NULL
  int rows;
  uint32_t cols, n_vec;
};

// Persistent: a row per warp or per CTA at a time.  Each thread keeps the
// column sums of its own pieces in registers over all its rows and leaves them
// in the workspace: one partial row per CTA.
template <typename T, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) bwd_kernel(const BwdArgs a) {
  __shared__ float s_red[2][2][32 * 3];
  pdl_enter();
  const uint32_t l = WARP ? threadIdx.x & 31 : threadIdx.x, L = WARP ? 32 : blockDim.x;
  const int slot = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int slots = WARP ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
  float c_pre[NV][VEC], c_post[NV][VEC], c_gate[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) c_pre[i][j] = c_post[i][j] = c_gate[i][j] = 0.f;
  const float inv_n = 1.f / (float)a.cols;
  int par = 0;
  for (long long row = slot; row < a.rows; row += slots, par ^= 1) {
    Raw<T, VEC> ry[NV] = {}, rh[NV] = {}, rdh[NV] = {}, rdx[NV] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t v = l + i * L;
      if (v < a.n_vec) {
        if (a.y) ry[i] = load_raw<T, VEC>((const T *)a.y + (size_t)row * a.ld_y, v);
        if (a.dxn) rh[i] = load_raw<T, VEC>((const T *)a.h + (size_t)row * a.ld_h, v);
        if (a.dh) rdh[i] = load_raw<T, VEC>((const T *)a.dh + (size_t)row * a.ld_dh, v);
        if (a.dxn) rdx[i] = load_raw<T, VEC>((const T *)a.dxn + (size_t)row * a.ld_dx, v);
      }
    }
    float s[3] = {0.f, 0.f, 0.f};  // sum y^2, sum h^2, sum u h
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t v = l + i * L;
      float e[VEC];
      if (a.post_w) {
        unpack<T, VEC>(ry[i], e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[0] = fmaf(e[j], e[j], s[0]);
      }
      if (a.dxn && v < a.n_vec) {
        float d[VEC], w[VEC];
        unpack<T, VEC>(rh[i], e);
        unpack<T, VEC>(rdx[i], d);
        load_param<VEC>(a.pre_w, v, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s[1] = fmaf(e[j], e[j], s[1]);
          s[2] = fmaf(d[j] * w[j], e[j], s[2]);
        }
      }
    }
    row_sum<WARP, 3>(s, s_red[par][0]);
    const float r_y = a.post_w ? 1.f / sqrtf(s[0] * inv_n + a.eps) : 1.f;
    const float r_h = 1.f / sqrtf(s[1] * inv_n + a.eps);
    const float m_h = s[2] * inv_n * r_h * r_h;
    const float gt = a.gate_kind == FFN_B200_GATE_TOKEN ? __ldg(a.gate + row) : 1.f;
    // g, its part of the residual, and the branch's sums
    float g[NV][VEC];
    float q[2] = {0.f, 0.f};  // sum v y, sum g b
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t v = l + i * L;
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[i][j] = 0.f;
      if (v < a.n_vec) {
        if (a.dh) unpack<T, VEC>(rdh[i], g[i]);
        if (a.dxn) {
          float e[VEC], d[VEC], w[VEC];
          unpack<T, VEC>(rh[i], e);
          unpack<T, VEC>(rdx[i], d);
          load_param<VEC>(a.pre_w, v, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            g[i][j] = fmaf(r_h, fmaf(d[j], w[j], -e[j] * m_h), g[i][j]);
            c_pre[i][j] = fmaf(d[j], e[j] * r_h, c_pre[i][j]);
          }
        }
        if (a.dres) {
          float o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = a.alpha * g[i][j];
          store_vec<T, VEC>((T *)a.dres + (size_t)row * a.ld_dr, v, o);
        }
        if (a.y) {
          float e[VEC], w[VEC], gc[VEC];
          unpack<T, VEC>(ry[i], e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) w[j] = 1.f, gc[j] = gt;
          if (a.post_w) load_param<VEC>(a.post_w, v, w);
          if (a.gate_kind == FFN_B200_GATE_CHANNEL) load_param<VEC>(a.gate, v, gc);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float yn = e[j] * r_y, bg = a.beta * g[i][j];
            c_gate[i][j] = fmaf(bg, yn * w[j], c_gate[i][j]);
            q[1] = fmaf(bg, yn * w[j], q[1]);
            const float db = bg * gc[j];
            c_post[i][j] = fmaf(db, yn, c_post[i][j]);
            g[i][j] = db * w[j];  // v
            q[0] = fmaf(g[i][j], e[j], q[0]);
          }
        }
      }
    }
    if (!a.y) continue;
    row_sum<WARP, 2>(q, s_red[par][1]);
    if (a.dgate_tok && l == 0) a.dgate_tok[row] = q[1];
    if (a.dy) {
      const float m_y = a.post_w ? q[0] * inv_n * r_y * r_y : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t v = l + i * L;
        if (v < a.n_vec) {
          float e[VEC];
          unpack<T, VEC>(ry[i], e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) e[j] = r_y * fmaf(-e[j], m_y, g[i][j]);
          store_vec<T, VEC>((T *)a.dy + (size_t)row * a.ld_dy, v, e);
        }
      }
    }
  }
  if (WARP && (a.part_pre || a.part_post || a.part_gate)) {
    // the CTA's eight warps add up in warp order; warp 7 then holds
    // their sums
    extern __shared__ float s_col[];  // [3][cols]
    for (int w = 0; w < 8; ++w) {
      if ((int)(threadIdx.x >> 5) == w) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const uint32_t v = l + i * L;
          if (v >= a.n_vec) continue;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float *at = s_col + (size_t)v * VEC + j;
            if (w) {
              c_pre[i][j] += at[0];
              c_post[i][j] += at[a.cols];
              c_gate[i][j] += at[2 * a.cols];
            }
            at[0] = c_pre[i][j], at[a.cols] = c_post[i][j], at[2 * a.cols] = c_gate[i][j];
          }
        }
      }
      __syncthreads();
    }
    if (threadIdx.x >> 5 != 7) return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t v = l + i * L;
    if (v >= a.n_vec) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const size_t at = (size_t)blockIdx.x * a.cols + (size_t)v * VEC + j;
      if (a.part_pre) a.part_pre[at] = c_pre[i][j];
      if (a.part_post) a.part_post[at] = c_post[i][j];
      if (a.part_gate) a.part_gate[at] = c_gate[i][j];
    }
  }
}

// Column sums of the partial rows, 32 columns a CTA: warp w adds every 8th row
// in order, then the eight sums are added in warp order.
struct ColArgs {
  const float *part[3];
  float *out[3];
  int parts;
  uint32_t cols;
};
__global__ void __launch_bounds__(256) colsum_kernel(const ColArgs a) {
  __shared__ float s[8][32];
  pdl_enter();
  const float *p = a.part[blockIdx.y];
  if (!p) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < a.cols) {
#pragma unroll 8
    for (int r = warp; r < a.parts; r += 8) sum += p[(size_t)r * a.cols + c];
  }
  s[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < a.cols) {
    for (int w = 1; w < 8; ++w) sum += s[w][lane];
    a.out[blockIdx.y][c] = sum;
  }
}

// ------------------------------------------------------------------ launch
// Short rows (up to 128 pieces of 16 bytes, or 512 single elements) take a
// warp each, longer ones a CTA of just enough threads.
struct Shape {
  bool warp;
  int nv, threads;
};
Shape shape_of(uint32_t n_vec, int vec) {
  if (vec > 1) {
    if (n_vec <= 128) return {true, 4, 256};
    const int nv = n_vec <= 2048 ? 2 : 4;
    return {false, nv, (int)(((n_vec + nv - 1) / nv + 31) / 32 * 32)};
  }
  if (n_vec <= 512) return {true, 16, 256};
  return {false, 16, (int)(((n_vec + 15) / 16 + 31) / 32 * 32)};
}

template <typename T, int VEC>
int launch_fwd(FwdArgs &a, cudaStream_t st) {
  a.n_vec = a.cols / VEC;
  const Shape s = shape_of(a.n_vec, VEC);
  const int grid = s.warp ? (a.rows + 7) / 8 : a.rows;
#define FFN_GO(NV, W) FFN_LAUNCH_PDL(FFN_B200_K_NORM, st, "block_norm", (fwd_kernel<T, VEC, NV, W>), grid, s.threads, 0, a)
  if constexpr (VEC > 1) {
    if (s.warp) FFN_GO(4, true);
    else if (s.nv == 2) FFN_GO(2, false);
    else FFN_GO(4, false);
  } else {
    if (s.warp) FFN_GO(16, true);
    else FFN_GO(16, false);
  }
#undef FFN_GO
  return 0;
}

int bwd_slots(size_t rows, uint32_t n_vec, int vec, int sms) {  // partial rows
  const Shape s = shape_of(n_vec, vec);
  if (s.warp) return (int)std::min<size_t>((rows + 7) / 8, (size_t)sms * 2);
  return (int)std::min<size_t>(rows, (size_t)sms * std::max(1, 1024 / s.threads));
}

template <typename T, int VEC>
int launch_bwd(BwdArgs &a, int slots, cudaStream_t st) {
  a.n_vec = a.cols / VEC;
  const Shape s = shape_of(a.n_vec, VEC);
  const size_t smem = s.warp ? 3 * a.cols * sizeof(float) : 0;  // 12 KB at most
#define FFN_GO(NV, W) FFN_LAUNCH_PDL(FFN_B200_K_NORM, st, "block_norm_bwd", (bwd_kernel<T, VEC, NV, W>), slots, s.threads, smem, a)
  if constexpr (VEC > 1) {
    if (s.warp) FFN_GO(4, true);
    else if (s.nv == 2) FFN_GO(2, false);
    else FFN_GO(4, false);
  } else {
    if (s.warp) FFN_GO(16, true);
    else FFN_GO(16, false);
  }
#undef FFN_GO
  return 0;
}

int check_desc(const char *what, const ffn_b200_block_norm_desc *d) {
  const std::string w(what);
  if (!d) return fail(FFN_B200_EINVAL, w + ": null descriptor");
  if (!dtype_ok(d->dtype)) return fail(FFN_B200_EINVAL, w + ": unknown dtype");
  if (d->cols == 0 || d->cols > (size_t)kMaxCols) return fail(FFN_B200_EUNSUP, w + ": cols must be in 1..16384");
  if (d->rows > 0x7fffffffu) return fail(FFN_B200_EINVAL, w + ": too many rows");
  if (d->gate_kind != FFN_B200_GATE_NONE && d->gate_kind != FFN_B200_GATE_CHANNEL && d->gate_kind != FFN_B200_GATE_TOKEN)
    return fail(FFN_B200_EINVAL, w + ": unknown gate_kind");
  if ((d->gate_kind != FFN_B200_GATE_NONE) != (d->gate != nullptr))
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

// The workspace does not depend on the pointers' alignment: the larger of both forms.
size_t ffn_b200_block_norm_bwd_ws_bytes(const ffn_b200_block_norm_desc *d) {
  using namespace ffn::bn;
  if (!d || d->cols == 0 || d->cols > (size_t)kMaxCols || !dtype_ok(d->dtype)) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    dev = -1;
  }
  const int sms = sm_count_of(dev), vec = (int)(16 / dtype_bytes(d->dtype));
  const int wide = d->cols % vec == 0 ? bwd_slots(d->rows, (uint32_t)(d->cols / vec), vec, sms) : 0;
  const int slots = std::max(wide, bwd_slots(d->rows, (uint32_t)d->cols, 1, sms));
  return (size_t)slots * d->cols * 3 * sizeof(float) + 16;
}

int ffn_b200_block_norm_bwd(const ffn_b200_block_norm_desc *d, const void *y, size_t ld_y, const void *h, size_t ld_h,
                            const void *dh, size_t ld_dh, const void *dxn, size_t ld_dxn, void *dresidual, size_t ld_dres,
                            void *dy, size_t ld_dy, float *dpost_w, float *dgate, float *dpre_w, void *ws, size_t ws_bytes,
                            void *stream) {
  using namespace ffn::bn;
  if (int rc = check_desc("block_norm_bwd", d)) return rc;
  if ((dpost_w && !d->post_w) || (dgate && !d->gate))
    return fail(FFN_B200_EINVAL, "block_norm_bwd: a gradient of a parameter that is not there");
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
  a.y = branch ? y : nullptr, a.h = h, a.dh = dh, a.dxn = dxn;
  a.ld_y = ld_y, a.ld_h = ld_h, a.ld_dh = ld_dh, a.ld_dx = ld_dxn, a.ld_dr = ld_dres, a.ld_dy = ld_dy;
  a.post_w = branch ? d->post_w : nullptr, a.gate = d->gate, a.pre_w = d->pre_w;
  a.gate_kind = d->gate_kind;
  a.alpha = d->alpha, a.beta = d->beta, a.eps = d->eps;
  a.dres = dresidual, a.dy = dy;
  a.dgate_tok = d->gate_kind == FFN_B200_GATE_TOKEN ? dgate : nullptr;
  a.rows = (int)d->rows;
  a.cols = (uint32_t)d->cols;
  const bool v16 = d->cols * es % 16 == 0 && rows16(a.y, ld_y, es) && rows16(dxn ? h : nullptr, ld_h, es) &&
                   rows16(dh, ld_dh, es) && rows16(dxn, ld_dxn, es) && rows16(dresidual, ld_dres, es) &&
                   rows16(dy, ld_dy, es) && params16(d);
  int dev = 0;
  FFN_CUDA_TRY(cudaGetDevice(&dev));
  const int vec = v16 ? (int)(16 / es) : 1;
  const int slots = bwd_slots(d->rows, (uint32_t)(d->cols / vec), vec, sm_count_of(dev));
  const size_t plane = (size_t)slots * d->cols;
  const bool any = dpre_w || dpost_w || chan;
  if (any) {
    if (!ws || (uintptr_t)ws % 4) return fail(FFN_B200_EINVAL, "block_norm_bwd: the workspace is null or misaligned");
    if (ws_bytes < ffn_b200_block_norm_bwd_ws_bytes(d)) return fail(FFN_B200_ENOSPC, "block_norm_bwd: workspace too small");
  }
  float *part = (float *)ws;
  if (dpre_w) a.part_pre = part;
  if (dpost_w) a.part_post = part + plane;
  if (chan) a.part_gate = part + 2 * plane;
  int rc;
  if (d->dtype == FFN_B200_DT_F32) rc = v16 ? launch_bwd<float, 4>(a, slots, st) : launch_bwd<float, 1>(a, slots, st);
  else if (d->dtype == FFN_B200_DT_BF16) rc = v16 ? launch_bwd<__nv_bfloat16, 8>(a, slots, st) : launch_bwd<__nv_bfloat16, 1>(a, slots, st);
  else rc = v16 ? launch_bwd<__half, 8>(a, slots, st) : launch_bwd<__half, 1>(a, slots, st);
  if (rc || !any) return rc;
  ColArgs c{};
  c.part[0] = a.part_pre, c.part[1] = a.part_post, c.part[2] = a.part_gate;
  c.out[0] = dpre_w, c.out[1] = dpost_w, c.out[2] = dgate;
  c.parts = slots;
  c.cols = a.cols;
  FFN_LAUNCH_PDL(FFN_B200_K_NORM, st, "colsum_kernel", colsum_kernel, dim3((a.cols + 31) / 32, 3), 256, 0, c);
  return 0;
}

}  // extern "C"
