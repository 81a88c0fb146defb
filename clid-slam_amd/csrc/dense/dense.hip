// The dense operators of include/clid_dense.h: a first form that is right for every size, type and layout.  One 64 x 64 tile per
// block, fp32 FMAs from LDS, operands read element by element through (row, column) strides.
#include "dense.hpp"

namespace clid_dense {

constexpr int kT = 64, kStep = 16;

// out(m, n) = sum_k a(m, k) b(n, k); T of the operands, each with its strides; a row m of `a` (or a step k, where rows are the
// contraction) whose target is `ignore` is read as zeros.
struct Gemm {
  const void *a, *b;
  int64_t a_row, a_k, b_row, b_k;
  int64_t m, n, k;
  const int64_t* target;
  int64_t ignore;
  int mask_k;  // the targets belong to k (else to m)
};

template <typename TA, typename TB>
__device__ __forceinline__ void tile(const Gemm& g, int64_t m0, int64_t n0, float (&acc)[4][4]) {
  __shared__ float sa[kStep][kT + 4], sb[kStep][kT + 4];
  const TA* a = (const TA*)g.a;
  const TB* b = (const TB*)g.b;
  const int t = threadIdx.x, tm = (t >> 4) * 4, tn = (t & 15) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (int64_t k0 = 0; k0 < g.k; k0 += kStep) {
    __syncthreads();
    for (int e = t; e < kT * kStep; e += 256) {
      // neighbouring threads along the operand's contiguous direction
      const int ar = g.a_k == 1 ? e / kStep : e % kT, ak = g.a_k == 1 ? e % kStep : e / kT;
      const int br = g.b_k == 1 ? e / kStep : e % kT, bk = g.b_k == 1 ? e % kStep : e / kT;
      float va = 0.f, vb = 0.f;
      if (m0 + ar < g.m && k0 + ak < g.k && !(g.target && !g.mask_k && g.target[m0 + ar] == g.ignore))
        va = up(a[(m0 + ar) * g.a_row + (k0 + ak) * g.a_k]);
      if (n0 + br < g.n && k0 + bk < g.k && !(g.target && g.mask_k && g.target[k0 + bk] == g.ignore))
        vb = up(b[(n0 + br) * g.b_row + (k0 + bk) * g.b_k]);
      sa[ak][ar] = va;
      sb[bk][br] = vb;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][tm + i], sb[k][tn + j], acc[i][j]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_linear(Gemm g, const T* bias, const T* res, int64_t ldr, T* y, T* z_out, int act) {
  float acc[4][4];
  const int64_t tn = (g.n + kT - 1) / kT, m0 = blockIdx.x / tn * kT, n0 = blockIdx.x % tn * kT;
  tile<T, T>(g, m0, n0, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + (threadIdx.x >> 4) * 4 + i, n = n0 + (threadIdx.x & 15) * 4 + j;
      if (m >= g.m || n >= g.n) continue;
      const float z = acc[i][j] + (bias ? up(bias[n]) : 0.f);
      if (z_out) z_out[m * g.n + n] = keep_z<T>(z);
      y[m * g.n + n] = down<T>(act_value(z, act) + (res ? up(res[m * ldr + n]) : 0.f));
    }
}

// out = alpha * sum (+ what `add` holds): TO fp32 or the operands' type
template <typename TA, typename TB, typename TO>
__global__ void __launch_bounds__(256) k_product(Gemm g, const float* add, const float* alpha, TO* out) {
  float acc[4][4];
  const int64_t tn = (g.n + kT - 1) / kT, m0 = blockIdx.x / tn * kT, n0 = blockIdx.x % tn * kT;
  tile<TA, TB>(g, m0, n0, acc);
  const float s = alpha ? *alpha : 1.f;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + (threadIdx.x >> 4) * 4 + i, n = n0 + (threadIdx.x & 15) * 4 + j;
      if (m < g.m && n < g.n) out[m * g.n + n] = down<TO>(s * acc[i][j] + (add ? add[m * g.n + n] : 0.f));
    }
}

template <typename T>
__global__ void k_dz(const T* dy, int64_t lddy, const T* z, int64_t rows, int n, int act, float* dz) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = i / n;
    dz[i] = up(dy[m * lddy + (i - m * n)]) * (z ? act_slope(up(z[i]), act) : 1.f);
  }
}

// sum over rows, one column per thread of x, rows over y
template <typename T>
__global__ void k_colsum(const float* v, int64_t rows, int n, const float* alpha, T* out) {
  __shared__ float part[4][64];
  const int c = blockIdx.x * 64 + threadIdx.x;
  float s = 0.f;
  if (c < n)
    for (int64_t m = threadIdx.y; m < rows; m += 4) s += v[m * n + c];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < n)
    out[c] = down<T>((alpha ? *alpha : 1.f) * (part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x]));
}

// statistics of the tile's columns for each of its rows -> part[m][column tile]; the target's z -> zt[m]
template <typename T>
__global__ void __launch_bounds__(256) k_stat(Gemm g, const T* bias, const int64_t* target, Stat* part, float* zt) {
  float acc[4][4];
  const int64_t tn = (g.n + kT - 1) / kT, m0 = blockIdx.x / tn * kT, n0 = blockIdx.x % tn * kT;
  tile<T, T>(g, m0, n0, acc);
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + (threadIdx.x >> 4) * 4 + i;
    Stat s = {neg_inf(), 0.f, 0x7fffffff};
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + (threadIdx.x & 15) * 4 + j;
      if (n >= g.n || m >= g.m) continue;
      const float z = acc[i][j] + (bias ? up(bias[n]) : 0.f);
      s = join(s, {z, 0.f, (int)n});
      if (target && target[m] == n) zt[m] = z;
    }
    for (int d = 1; d < 16; d <<= 1)
      s = join(s, {__shfl_xor(s.m, d, 64), __shfl_xor(s.r, d, 64), __shfl_xor(s.at, d, 64)});
    if ((threadIdx.x & 15) == 0 && m < g.m) part[m * tn + blockIdx.x % tn] = s;
  }
}

__global__ void k_label(const Stat* part, int tiles, int64_t rows, int64_t* label, float* log_prob) {
  const int64_t m = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (m >= rows) return;
  Stat s = part[m * tiles];
  for (int i = 1; i < tiles; ++i) s = join(s, part[m * tiles + i]);
  label[m] = s.at;
  log_prob[m] = s.m == neg_inf() ? __builtin_nanf("") : -log1pf(s.r);
}

__global__ void k_loss_rows(const Stat* part, int tiles, const float* zt, const int64_t* target, int64_t rows, int n, int64_t ignore,
                            float4* stat, float* loss_none) {
  const int64_t m = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (m >= rows) return;
  const int64_t t = target[m];
  float4 o = {0.f, 0.f, 0.f, 0.f};
  if (t != ignore) {
    Stat s = part[m * tiles];
    for (int i = 1; i < tiles; ++i) s = join(s, part[m * tiles + i]);
    const float loss = t >= 0 && t < n ? (s.m - zt[m]) + log1pf(s.r) : __builtin_nanf("");
    o = {s.m, 1.f / (1.f + s.r), expm1f(-loss), loss};
  }
  stat[m] = o;
  if (loss_none) loss_none[m] = o.w;
}

// one block: the sum of the rows' losses, how many count, and the reduced loss
__global__ void __launch_bounds__(1024) k_loss_total(const float4* stat, const int64_t* target, int64_t rows, int64_t ignore, int reduction,
                                                     float* total, float* loss_out) {
  __shared__ double ps[16];
  __shared__ int pc[16];
  double s = 0.0;
  int c = 0;
  for (int64_t m = threadIdx.x; m < rows; m += 1024) {
    const bool on = target[m] != ignore;
    s += on ? (double)stat[m].w : 0.0;
    c += on;
  }
  for (int d = 32; d; d >>= 1) {
    s += __shfl_xor(s, d, 64);
    c += __shfl_xor(c, d, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    ps[threadIdx.x >> 6] = s;
    pc[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    c = 0;
    for (int i = 0; i < 16; ++i) {
      s += ps[i];
      c += pc[i];
    }
    total[0] = (float)s;
    total[1] = (float)c;
    if (reduction == CLID_REDUCE_MEAN) loss_out[0] = c ? (float)(s / c) : 0.f;
    if (reduction == CLID_REDUCE_SUM) loss_out[0] = (float)s;
  }
}

// dz of a piece of the vocabulary (columns v0 .. v0 + g.n)
template <typename T>
__global__ void __launch_bounds__(256) k_ce_dz(Gemm g, const T* bias, int64_t v0, const int64_t* target, int64_t ignore, const float4* stat,
                                               const float* grad, int reduction, const float* total, float* dz) {
  float acc[4][4];
  const int64_t tn = (g.n + kT - 1) / kT, m0 = blockIdx.x / tn * kT, n0 = blockIdx.x % tn * kT;
  tile<T, T>(g, m0, n0, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + (threadIdx.x >> 4) * 4 + i, n = n0 + (threadIdx.x & 15) * 4 + j;
      if (m >= g.m || n >= g.n) continue;
      const int64_t t = target[m];
      float v = 0.f;
      if (t != ignore) {
        const float4 s = stat[m];
        const float gr = reduction == CLID_REDUCE_NONE ? grad[m] : reduction == CLID_REDUCE_MEAN ? grad[0] / total[1] : grad[0];
        const float z = acc[i][j] + (bias ? up(bias[n]) : 0.f);
        v = gr * (t == v0 + n ? s.z : (s.w != s.w ? s.w : expf(z - s.x) * s.y));
      }
      dz[m * g.n + n] = v;
    }
}

inline dim3 tiles_of(int64_t m, int64_t n) { return dim3((unsigned)((n + kT - 1) / kT * ((m + kT - 1) / kT))); }

}  // namespace clid_dense

using namespace clid_dense;

#define BY_DTYPE(dtype, ...)                                   \
  do {                                                         \
    if ((dtype) == CLID_F32) { using T = float; __VA_ARGS__ }  \
    else if ((dtype) == CLID_BF16) { using T = bf16; __VA_ARGS__ } \
    else { using T = f16; __VA_ARGS__ }                        \
  } while (0)

static int bad(const char* what, const char* why) {
  clid_set_error("%s: %s", what, why);
  return CLID_E_ARG;
}
static bool dtype_ok(int d) { return d == CLID_F32 || d == CLID_BF16 || d == CLID_F16; }

extern "C" int64_t clid_linear_workspace(const clid_linear_args* a) { return a ? 256 : CLID_E_ARG; }
extern "C" int clid_linear_fwd(const clid_linear_args* a, void* stream) {
  const char* me = "clid_linear_fwd";
  if (!a || !sizes_ok(a->rows, a->k, a->n) || !dtype_ok(a->dtype) || a->act < 0 || a->act > CLID_ACT_SILU) return bad(me, "bad argument");
  if (a->rows == 0) return CLID_OK;
  if (!a->x || !a->w || !a->y || a->ldx < a->k || a->ldw < a->k || (a->residual && a->ldr < a->n)) return bad(me, "bad pointer or row stride");
  BY_DTYPE(a->dtype, Gemm g = {a->x, a->w, a->ldx, 1, a->ldw, 1, a->rows, a->n, a->k, nullptr, 0, 0};
           hipLaunchKernelGGL(k_linear<T>, tiles_of(a->rows, a->n), dim3(256), 0, (hipStream_t)stream, g, (const T*)a->bias,
                              (const T*)a->residual, a->ldr, (T*)a->y, (T*)a->z_out, a->act););
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}

extern "C" int64_t clid_linear_bwd_workspace(const clid_linear_bwd_args* a) { return a ? up256(a->rows * a->n * 4) : CLID_E_ARG; }
extern "C" int clid_linear_bwd(const clid_linear_bwd_args* a, void* stream) {
  const char* me = "clid_linear_bwd";
  if (!a || !sizes_ok(a->rows, a->k, a->n) || !dtype_ok(a->dtype) || a->act < 0 || a->act > CLID_ACT_SILU) return bad(me, "bad argument");
  if (a->rows == 0) return bad(me, "no rows");
  if (!a->x || !a->w || !a->dy || a->ldx < a->k || a->ldw < a->k || a->lddy < a->n || (!a->z && a->act != CLID_ACT_NONE)) return bad(me, "bad pointer or row stride");
  if (!a->ws || a->ws_bytes < clid_linear_bwd_workspace(a)) return bad(me, "workspace too small");
  hipStream_t s = (hipStream_t)stream;
  float* dz = (float*)a->ws;
  const int64_t blocks = (a->rows * a->n + 255) / 256;
  BY_DTYPE(a->dtype, {
    hipLaunchKernelGGL(k_dz<T>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, (const T*)a->dy, a->lddy, (const T*)a->z, a->rows, a->n, a->act, dz);
    if (a->dx) {
      Gemm g = {dz, a->w, a->n, 1, 1, a->ldw, a->rows, a->k, a->n, nullptr, 0, 0};
      hipLaunchKernelGGL((k_product<float, T, T>), tiles_of(a->rows, a->k), dim3(256), 0, s, g, (const float*)nullptr, (const float*)nullptr, (T*)a->dx);
    }
    if (a->dw) {
      Gemm g = {dz, a->x, 1, a->n, 1, a->ldx, a->n, a->k, a->rows, nullptr, 0, 0};
      hipLaunchKernelGGL((k_product<float, T, T>), tiles_of(a->n, a->k), dim3(256), 0, s, g, (const float*)nullptr, (const float*)nullptr, (T*)a->dw);
    }
    if (a->db) hipLaunchKernelGGL(k_colsum<T>, dim3((a->n + 63) / 64), dim3(64, 4), 0, s, dz, a->rows, a->n, (const float*)nullptr, (T*)a->db);
  });
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}

static int64_t stat_bytes(int64_t rows, int32_t n) { return up256(rows * ((n + kT - 1) / kT) * (int64_t)sizeof(Stat)); }

extern "C" int64_t clid_ce_workspace(const clid_ce_args* a) { return a ? stat_bytes(a->rows, a->n) + up256(a->rows * 4) : CLID_E_ARG; }
static bool ce_ok(const clid_ce_args* a) {
  return a && sizes_ok(a->rows, a->k, a->n) && dtype_ok(a->dtype) && a->reduction >= 0 && a->reduction <= CLID_REDUCE_SUM;
}
extern "C" int clid_ce_fwd(const clid_ce_args* a, void* stream) {
  const char* me = "clid_ce_fwd";
  if (!ce_ok(a)) return bad(me, "bad argument");
  if (!a->total || (a->rows && (!a->x || !a->w || !a->target || !a->stat)) || (!a->loss_out && !(a->reduction == CLID_REDUCE_NONE && a->rows == 0)) ||
      a->ldx < a->k || a->ldw < a->k) return bad(me, "bad pointer or row stride");
  if (a->rows && (!a->ws || a->ws_bytes < clid_ce_workspace(a))) return bad(me, "workspace too small");
  hipStream_t s = (hipStream_t)stream;
  if (a->rows) {
    Stat* part = (Stat*)a->ws;
    float* zt = (float*)((char*)a->ws + stat_bytes(a->rows, a->n));
    const int tiles = (a->n + kT - 1) / kT;
    BY_DTYPE(a->dtype, Gemm g = {a->x, a->w, a->ldx, 1, a->ldw, 1, a->rows, a->n, a->k, a->target, a->ignore_index, 0};
             hipLaunchKernelGGL(k_stat<T>, tiles_of(a->rows, a->n), dim3(256), 0, s, g, (const T*)a->bias, a->target, part, zt););
    hipLaunchKernelGGL(k_loss_rows, dim3((unsigned)((a->rows + 255) / 256)), dim3(256), 0, s, part, tiles, zt, a->target, a->rows, a->n,
                       a->ignore_index, (float4*)a->stat, a->reduction == CLID_REDUCE_NONE ? a->loss_out : nullptr);
  }
  hipLaunchKernelGGL(k_loss_total, dim3(1), dim3(1024), 0, s, (const float4*)a->stat, a->target, a->rows, a->ignore_index, a->reduction, a->total, a->loss_out);
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}

// columns of the vocabulary per piece: 256 MB of dz
static int64_t piece_of(const clid_ce_args* a) {
  int64_t p = (int64_t(64) << 20) / (a->rows > 0 ? a->rows : 1) / 64 * 64;
  if (p < 64) p = 64;
  return p < a->n ? p : a->n;
}
extern "C" int64_t clid_ce_bwd_workspace(const clid_ce_args* a) {
  return a ? up256(a->rows * piece_of(a) * 4) + up256(a->rows * a->k * 4) : CLID_E_ARG;
}
extern "C" int clid_ce_bwd(const clid_ce_args* a, void* stream) {
  const char* me = "clid_ce_bwd";
  if (!ce_ok(a)) return bad(me, "bad argument");
  if (a->rows == 0) return bad(me, "no rows");
  if (!a->x || !a->w || !a->target || !a->stat || !a->total || !a->g || a->ldx < a->k || a->ldw < a->k) return bad(me, "bad pointer or row stride");
  if (!a->ws || a->ws_bytes < clid_ce_bwd_workspace(a)) return bad(me, "workspace too small");
  hipStream_t s = (hipStream_t)stream;
  const int64_t piece = piece_of(a);
  float* dz = (float*)a->ws;
  float* sum = (float*)((char*)a->ws + up256(a->rows * piece * 4));
  BY_DTYPE(a->dtype, {
    for (int64_t v0 = 0; v0 < a->n; v0 += piece) {
      const int64_t nv = a->n - v0 < piece ? a->n - v0 : piece;
      const T* w = (const T*)a->w + v0 * a->ldw;
      Gemm g = {a->x, w, a->ldx, 1, a->ldw, 1, a->rows, nv, a->k, a->target, a->ignore_index, 0};
      hipLaunchKernelGGL(k_ce_dz<T>, tiles_of(a->rows, nv), dim3(256), 0, s, g, a->bias ? (const T*)a->bias + v0 : nullptr, v0, a->target,
                         a->ignore_index, (const float4*)a->stat, a->g, a->reduction, a->total, dz);
      if (a->dx) {
        Gemm d = {dz, w, nv, 1, 1, a->ldw, a->rows, a->k, nv, nullptr, 0, 0};
        const float* before = v0 ? sum : nullptr;
        if (v0 + nv < a->n)
          hipLaunchKernelGGL((k_product<float, T, float>), tiles_of(a->rows, a->k), dim3(256), 0, s, d, before, (const float*)nullptr, sum);
        else
          hipLaunchKernelGGL((k_product<float, T, T>), tiles_of(a->rows, a->k), dim3(256), 0, s, d, before, (const float*)nullptr, (T*)a->dx);
      }
      if (a->dw) {
        Gemm d = {dz, a->x, 1, nv, 1, a->ldx, nv, a->k, a->rows, a->target, a->ignore_index, 1};
        hipLaunchKernelGGL((k_product<float, T, T>), tiles_of(nv, a->k), dim3(256), 0, s, d, (const float*)nullptr, (const float*)nullptr, (T*)a->dw + v0 * a->k);
      }
      if (a->db) hipLaunchKernelGGL(k_colsum<T>, dim3((unsigned)((nv + 63) / 64)), dim3(64, 4), 0, s, dz, a->rows, (int)nv, (const float*)nullptr, (T*)a->db + v0);
    }
  });
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}

extern "C" int64_t clid_label_workspace(const clid_label_args* a) { return a ? stat_bytes(a->rows, a->n) : CLID_E_ARG; }
extern "C" int clid_label_fwd(const clid_label_args* a, void* stream) {
  const char* me = "clid_label_fwd";
  if (!a || !sizes_ok(a->rows, a->k, a->n) || !dtype_ok(a->dtype)) return bad(me, "bad argument");
  if (a->rows == 0) return CLID_OK;
  if (!a->x || !a->w || !a->label || !a->log_prob || a->ldx < a->k || a->ldw < a->k) return bad(me, "bad pointer or row stride");
  if (!a->ws || a->ws_bytes < clid_label_workspace(a)) return bad(me, "workspace too small");
  Stat* part = (Stat*)a->ws;
  BY_DTYPE(a->dtype, Gemm g = {a->x, a->w, a->ldx, 1, a->ldw, 1, a->rows, a->n, a->k, nullptr, 0, 0};
           hipLaunchKernelGGL(k_stat<T>, tiles_of(a->rows, a->n), dim3(256), 0, (hipStream_t)stream, g, (const T*)a->bias, (const int64_t*)nullptr, part, (float*)nullptr););
  hipLaunchKernelGGL(k_label, dim3((unsigned)((a->rows + 255) / 256)), dim3(256), 0, (hipStream_t)stream, part, (a->n + kT - 1) / kT, a->rows, a->label, a->log_prob);
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}
