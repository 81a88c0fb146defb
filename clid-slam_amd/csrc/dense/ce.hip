// Softmax cross entropy of a class head and the class of each row, without the logits (include/clid_dense.h).
//
// Rows that count are brought together first (their numbers in `order`, the rows themselves copied without gaps), so a row that does
// not count costs nothing in the products and what it holds reaches none of them.
//
// Bound by its products, one forward (its sums become statistics in the tile's registers) and three backward, z made again among them: 8192 x 2048
// -> 65536 bf16 with 1 row in 10 ignored 7.0 ms, 1060 to 1210 TFLOP/s each; 2048 x 1024 -> 32000 fp32 2.8 ms, 173 to 205.  The rest (bringing rows
// together, joining strips, scale) is under 1 % there; with few rows and many classes it is not: 333 x 768 -> 50021 fp16 per row 72 us, 54 of them the
// product and 17 the join of 782 strips (k_loss_rows, 16 rows a block).
#include "stage.hpp"

using namespace clid_dense;

namespace {

constexpr int kRowsPer = 8192;  // rows a block of k_count / k_order looks at, 8 a thread
constexpr int kJoinRows = 16;   // rows a block of k_loss_rows joins

__device__ __forceinline__ int block_scan(int v, int* total) {  // exclusive, 1024 threads
  __shared__ int wsum[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(s, d, 64);
    if (lane >= d) s += o;
  }
  if (lane == 63) wsum[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < 16; ++i) {
    if (i < wave) before += wsum[i];
    all += wsum[i];
  }
  *total = all;
  return before + s - v;
}

// counts[block] = rows of the block that count
__global__ void __launch_bounds__(1024) k_count(const int64_t* target, int64_t rows, int64_t ignore, int* counts) {
  int c = 0;
  const int64_t at = (int64_t)blockIdx.x * kRowsPer + threadIdx.x * 8;
  for (int i = 0; i < 8; ++i) c += at + i < rows && target[at + i] != ignore;
  int total;
  block_scan(c, &total);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}
// order[0 ..) = the rows that count, in their order; order[rows] = how many; the others' loss
__global__ void __launch_bounds__(1024) k_order(const int64_t* target, int64_t rows, int64_t ignore, const int* counts, int32_t* order, float* loss_none) {
  const int64_t at = (int64_t)blockIdx.x * kRowsPer + threadIdx.x * 8;
  int before = 0, total;
  for (int b = threadIdx.x; b < (int)blockIdx.x; b += 1024) before += counts[b];
  block_scan(before, &total);
  before = total;
  __syncthreads();
  int on[8], c = 0;
  for (int i = 0; i < 8; ++i) {
    on[i] = at + i < rows && target[at + i] != ignore;
    c += on[i];
    if (loss_none && at + i < rows && !on[i]) loss_none[at + i] = 0.f;
  }
  int to = before + block_scan(c, &total);
  for (int i = 0; i < 8; ++i)
    if (on[i]) order[to++] = (int32_t)(at + i);
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) order[rows] = before + total;
}

// blocks of at most 1024 threads that one launch takes (2^32 threads); what is left they walk
constexpr int64_t kMostJoins = int64_t(1) << 21;

// a row's strips joined: 16 rows a block and turn, 32 threads a row; the block's sum of losses
__global__ void __launch_bounds__(512) k_loss_rows(const float2* part, int strips, const float* zt, const int64_t* target, const int32_t* order,
                                                   int64_t rows, int n, float4* stat, float* loss_none, double* sums) {
  __shared__ float pm[32][kJoinRows], pr[32][kJoinRows];
  const int64_t live = order[rows];
  const int row = threadIdx.x % kJoinRows, g = threadIdx.x / kJoinRows;
  double sum = 0.0;
  for (int64_t j0 = (int64_t)blockIdx.x * kJoinRows; j0 < live; j0 += (int64_t)gridDim.x * kJoinRows) {
    const int64_t j = j0 + row;
    Stat s = {neg_inf(), 0.f, 0};
    if (j < live)
#pragma unroll 4
      for (int i = g; i < strips; i += 32) {
        const float2 p = part[(int64_t)i * rows + j];
        s = join(s, {p.x, p.y, 0});
      }
    __syncthreads();  // the turn before has been read
    pm[g][row] = s.m;
    pr[g][row] = s.r;
    __syncthreads();
    if (g == 0 && j < live) {
      for (int i = 1; i < 32; ++i) s = join(s, {pm[i][row], pr[i][row], 0});
      const int64_t m = order[j], t = target[m];
      const float loss = t >= 0 && t < n ? (s.m - zt[j]) + log1pf(s.r) : __builtin_nanf("");
      stat[j] = {s.m, 1.f / (1.f + s.r), expm1f(-loss), loss};
      if (loss_none) loss_none[m] = loss;
      sum += loss;
    }
  }
  if (g) return;
  for (int d = kJoinRows / 2; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}
__global__ void __launch_bounds__(1024) k_loss_total(const double* sums, int blocks, const int32_t* live, int reduction, float* total, float* loss_out) {
  __shared__ double ps[16];
  double s = 0.0;
  for (int b = threadIdx.x; b < blocks; b += 1024) s += sums[b];
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
  if ((threadIdx.x & 63) == 0) ps[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int i = 0; i < 16; ++i) s += ps[i];
  const int c = live ? *live : 0;
  total[0] = (float)s;
  total[1] = (float)c;
  if (reduction == CLID_REDUCE_MEAN) loss_out[0] = c ? (float)(s / c) : 0.f;
  if (reduction == CLID_REDUCE_SUM) loss_out[0] = (float)s;
}

__global__ void __launch_bounds__(256) k_label_join(const float2* part, const int32_t* part_at, int strips, int64_t rows, int64_t* label, float* log_prob) {
  __shared__ float pm[16][16], pr[16][16];
  __shared__ int pa[16][16];
  const int row = threadIdx.x & 15, g = threadIdx.x >> 4;
  for (int64_t m0 = (int64_t)blockIdx.x * 16; m0 < rows; m0 += (int64_t)gridDim.x * 16) {
    const int64_t m = m0 + row;
    Stat s = {neg_inf(), 0.f, 0x7fffffff};
    if (m < rows)
      for (int i = g; i < strips; i += 16) {
        const float2 p = part[(int64_t)i * rows + m];
        s = join(s, {p.x, p.y, part_at[(int64_t)i * rows + m]});
      }
    __syncthreads();  // the turn before has been read
    pm[g][row] = s.m;
    pr[g][row] = s.r;
    pa[g][row] = s.at;
    __syncthreads();
    if (g || m >= rows) continue;
    for (int i = 1; i < 16; ++i) s = join(s, {pm[i][row], pr[i][row], pa[i][row]});
    label[m] = s.at;
    log_prob[m] = s.m == neg_inf() ? __builtin_nanf("") : -log1pf(s.r);
  }
}

// scale[0]: what dz is multiplied by as it is stored, scale[1]: what its products are multiplied by.  mean and sum: the one factor
// belongs to the products, and fp16's dz = p - onehot is stored times 2^10 so that small p keep their bits (|dz| <= 1).  none: the
// rows' factors go into dz, fp16's scaled by the power of two that brings the largest to at most 2^10; a row that does not count has no say in it,
// whatever its factor.  More than kTopRows rows are looked at by blocks of their own first (k_top: 64 -> 72 fp16 loss and gradients of 1048576 rows
// 1352 us, 2025 by the one block, of 32768 rows 111 and 113, of 16384 rows 78 and 77).  All blocks but the first: zeros for the
// rows of dx that do not count (one launch for both: 333 x 300 -> 200 fp32 loss and gradients 60.8 -> 58.9 us).
constexpr int64_t kTopRows = 16384;
__device__ __forceinline__ float largest(const float* g, const int64_t* target, int64_t ignore, int64_t from, int64_t rows, int64_t step) {
  float top = 0.f;
#pragma unroll 8
  for (int64_t m = from; m < rows; m += step) {
    const float v = fabsf(g[m]);
    top = v <= 3.4028235e38f && target[m] != ignore ? fmaxf(top, v) : top;
  }
  return top;
}
__device__ __forceinline__ float block_largest(float top) {  // 1024 threads; the first one's result
  __shared__ float ps[16];
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
  if ((threadIdx.x & 63) == 0) ps[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int i = 0; i < 16; ++i) top = fmaxf(top, ps[i]);
  return top;
}
__global__ void __launch_bounds__(1024) k_top(const float* g, const int64_t* target, int64_t ignore, int64_t rows, float* tops) {
  const float top = block_largest(largest(g, target, ignore, (int64_t)blockIdx.x * 1024 + threadIdx.x, rows, (int64_t)gridDim.x * 1024));
  if (threadIdx.x == 0) tops[blockIdx.x] = top;
}
template <typename T>
__global__ void __launch_bounds__(1024) k_scale(const float* g, const float* total, int64_t rows, int reduction, const float* tops, int n_tops, float* scale,
                                                const int64_t* target, int64_t ignore, int k, T* dx) {
  constexpr bool half = Kind<T>::F16;
  if (blockIdx.x) {
    for (int64_t m = (int64_t)(blockIdx.x - 1) * 4 + (threadIdx.x >> 8); m < rows; m += (int64_t)(gridDim.x - 1) * 4)
      if (target[m] == ignore)
        for (int c = threadIdx.x & 255; c < k; c += 256) dx[m * k + c] = down<T>(0.f);
    return;
  }
  if (reduction != CLID_REDUCE_NONE) {
    if (threadIdx.x == 0) {
      const float f = half ? 1024.f : 1.f;
      scale[0] = f;
      scale[1] = (reduction == CLID_REDUCE_MEAN ? g[0] / fmaxf(total[1], 1.f) : g[0]) / f;
    }
    return;
  }
  float top = 0.f;
  if (half) top = block_largest(n_tops ? (int)threadIdx.x < n_tops ? tops[threadIdx.x] : 0.f : largest(g, target, ignore, threadIdx.x, rows, 1024));
  if (threadIdx.x) return;
  int e = 0;
  if (top > 0.f) frexpf(top, &e);  // top < 2^e
  const int by = half && top > 0.f ? (10 - e > 100 ? 100 : 10 - e < -100 ? -100 : 10 - e) : 0;
  scale[0] = ldexpf(1.f, by);
  scale[1] = ldexpf(1.f, -by);
}

template <typename T, int SIZE> constexpr int strip_of() { return Tile<Kind<T>::NP, SIZE>::BN / Tile<Kind<T>::NP, SIZE>::WN; }
template <typename T>
int strip_width(int size) { return size == 2 ? strip_of<T, 2>() : size == 1 ? strip_of<T, 1>() : strip_of<T, 0>(); }

// rows of a wave
template <typename T, int SIZE> constexpr int run_of() { return Tile<Kind<T>::NP, SIZE>::BM / Tile<Kind<T>::NP, SIZE>::WM; }
template <typename T>
int run_rows(int size) { return size == 2 ? run_of<T, 2>() : size == 1 ? run_of<T, 1>() : run_of<T, 0>(); }

template <typename T, bool LABEL>
int launch_stat(const Product& g, int size, const T* bias, const int64_t* target, const int32_t* order, float2* part, int32_t* part_at, float* zt, hipStream_t s) {
  constexpr int NP = Kind<T>::NP;
  if (size == 2) return launch_one<T, 2, false, false>(g, EpiStat<T, Tile<NP, 2>::BN, strip_of<T, 2>(), LABEL>{bias, target, order, part, part_at, zt, g.m, g.n}, s);
  if (size == 1) return launch_one<T, 1, false, false>(g, EpiStat<T, Tile<NP, 1>::BN, strip_of<T, 1>(), LABEL>{bias, target, order, part, part_at, zt, g.m, g.n}, s);
  return launch_one<T, 0, false, false>(g, EpiStat<T, Tile<NP, 0>::BN, strip_of<T, 0>(), LABEL>{bias, target, order, part, part_at, zt, g.m, g.n}, s);
}
template <typename T>
int launch_dz(const Product& g, int size, const EpiDz<T, 0, Kind<T>::NP>& e, hipStream_t s) {
  constexpr int NP = Kind<T>::NP;
#define DZ(S) launch_one<T, S, false, false>(g, EpiDz<T, Tile<NP, S>::BN, NP>{e.bias, e.target, e.order, e.stat, e.scale, e.g, e.dz, e.sums, e.v0, e.n, e.ld}, s)
  return size == 2 ? DZ(2) : size == 1 ? DZ(1) : DZ(0);
#undef DZ
}

bool ce_ok(const clid_ce_args* a) {
  return a && sizes_ok(a->rows, a->k, a->n) && dtype_ok(a->dtype) && a->reduction >= 0 && a->reduction <= CLID_REDUCE_SUM;
}

// clid_ce_args.saved: the sum of the losses and how many rows count (fp32); the rows that count in their order, and in the place after the
// last how many there are; by place in that order: largest z, 1 / sum exp(z - largest), p_target - 1, loss
struct Saved {
  float* total;
  int32_t* order;
  float4* stat;
  int64_t bytes;
  explicit Saved(const clid_ce_args* a) {
    Ws ws(a->saved);
    total = (float*)ws.take(8);
    const bool lists = !is_narrow(a->k, a->n);
    order = (int32_t*)ws.take(lists ? (a->rows + 1) * 4 : 0);
    stat = (float4*)ws.take(lists ? a->rows * 16 : 0);
    bytes = ws.used;
  }
};

template <typename T>
struct CeFwd {
  Plan p;
  int strips, joins;
  char *x, *w, *counts, *part, *zt, *sums;
  int64_t bytes;
  explicit CeFwd(const clid_ce_args* a) {
    Ws ws(a->ws);
    p = plan<Kind<T>::NP>(a->rows, a->n, a->k, false);
    strips = (a->n + strip_width<T>(p.size) - 1) / strip_width<T>(p.size);
    const int64_t j = (a->rows + kJoinRows - 1) / kJoinRows;
    joins = (int)(j < kMostJoins ? j : kMostJoins);
    x = ws.take(stage_bytes<T>(a->x, a->ldx, a->rows, a->k, true));
    w = ws.take(stage_bytes<T>(a->w, a->ldw, a->n, a->k));
    counts = ws.take((a->rows + kRowsPer - 1) / kRowsPer * 4);
    part = ws.take((int64_t)strips * a->rows * 8);
    zt = ws.take(a->rows * 4);
    sums = ws.take((int64_t)joins * 8);
    bytes = ws.used;
  }
};

template <typename T>
int ce_fwd(const clid_ce_args* a, hipStream_t s) {
  const CeFwd<T> f(a);
  const Saved v(a);
  float* none = a->reduction == CLID_REDUCE_NONE ? a->loss_out : nullptr;
  if (a->rows) {
    const int blocks = (int)((a->rows + kRowsPer - 1) / kRowsPer);
    if (blocks > 1) hipLaunchKernelGGL(k_count, dim3(blocks), dim3(1024), 0, s, a->target, a->rows, a->ignore_index, (int*)f.counts);
    hipLaunchKernelGGL(k_order, dim3(blocks), dim3(1024), 0, s, a->target, a->rows, a->ignore_index, (const int*)f.counts, v.order, none);
    const int32_t* live = v.order + a->rows;
    const Staging x = staging<T>(a->x, a->ldx, a->rows, a->k, f.x, true, v.order, live), w = staging<T>(a->w, a->ldw, a->n, a->k, f.w);
    stage<T>(x, w, s);
    Product g = {staged<T>(x), staged<T>(w), a->rows, a->n, up8(a->k), live, 0, 1, 0, 0};
    const int rc = launch_stat<T, false>(g, f.p.size, (const T*)a->bias, a->target, v.order, (float2*)f.part, nullptr, (float*)f.zt, s);
    if (rc != CLID_OK) return rc;
    hipLaunchKernelGGL(k_loss_rows, dim3(f.joins), dim3(512), 0, s, (const float2*)f.part, f.strips, (const float*)f.zt, a->target, v.order, a->rows, a->n,
                       v.stat, none, (double*)f.sums);
  }
  hipLaunchKernelGGL(k_loss_total, dim3(1), dim3(1024), 0, s, (const double*)f.sums, f.joins, a->rows ? v.order + a->rows : nullptr, a->reduction, v.total, a->loss_out);
  return CLID_OK;
}

// Classes per piece: 512 MB of dz, in whole tiles, all pieces alike.  (8192 x 2048 -> 65536 bf16 and 2048 x 1024 -> 32000 fp32 loss and gradients
// with 128, 512, 2048 MB: 7.57, 7.59, 7.64 and 2.93, 2.74, 2.74 ms; 7000 x 512 -> 40000 fp16 in two of 20224 and 19776 classes: 1.46 ms, as 38144 and 1856: 1.64.)
template <typename T>
int64_t piece_of(const clid_ce_args* a) {
  int64_t p = (int64_t(512) << 20) / (2 * Kind<T>::NP * (a->rows > 0 ? a->rows : 1)) / 256 * 256;
  if (p < 256) p = 256;
  const int64_t pieces = (a->n + p - 1) / p, even = ((a->n + pieces - 1) / pieces + 255) / 256 * 256;
  return even < a->n ? even : a->n;
}

template <typename T>
struct CeBwd {
  int64_t piece, ld;
  Plan pz, px, pw;
  int runs, groups, share;  // db: partial sums, joined `share` at a time first where there are many (groups: 0 where not)
  int tops;                 // blocks of k_top
  char *x, *w, *dz, *sum, *part, *sums, *joined, *scale, *top;
  int64_t bytes;
  explicit CeBwd(const clid_ce_args* a) {
    constexpr int NP = Kind<T>::NP;
    Ws ws(a->ws);
    piece = piece_of<T>(a);
    ld = padded<T>(piece);
    pz = plan<NP>(a->rows, piece, a->k, false);
    px = plan<NP>(a->rows, a->k, piece, true);
    pw = plan<NP>(piece, a->k, a->rows, true);
    x = ws.take(stage_bytes<T>(a->x, a->ldx, a->rows, a->k, true));
    w = ws.take(stage_bytes<T>(a->w, a->ldw, a->n, a->k));
    dz = ws.take(NP * a->rows * ld * 2);
    sum = ws.take(a->dx && piece < a->n ? a->rows * a->k * 4 : 0);
    const int64_t bx = a->dx ? part_bytes(px, a->rows, a->k) : 0, bw = a->dw ? part_bytes(pw, piece, a->k) : 0;
    part = ws.take(bx > bw ? bx : bw);
    runs = (int)((a->rows + run_rows<T>(pz.size) - 1) / run_rows<T>(pz.size));
    share = runs <= 256 * 1024 ? 256 : (runs + 1023) / 1024;
    groups = runs > 1024 ? (runs + share - 1) / share : 0;
    sums = ws.take(a->db ? runs * piece * 4 : 0);
    joined = ws.take(a->db ? groups * piece * 4 : 0);
    scale = ws.take(8);
    const int64_t t = (a->rows + 2047) / 2048;
    tops = Kind<T>::F16 && a->reduction == CLID_REDUCE_NONE && a->rows > kTopRows ? (int)(t < 256 ? t : 256) : 0;
    top = ws.take(tops * 4);
    bytes = ws.used;
  }
};

template <typename T>
int ce_bwd(const clid_ce_args* a, hipStream_t s) {
  constexpr int NP = Kind<T>::NP;
  const CeBwd<T> f(a);
  const Saved v(a);
  const int32_t* live = v.order + a->rows;
  float* scale = (float*)f.scale;
  const int64_t clear = a->dx ? (a->rows + 3) / 4 : 0;
  if (f.tops) hipLaunchKernelGGL(k_top, dim3(f.tops), dim3(1024), 0, s, a->g, a->target, a->ignore_index, a->rows, (float*)f.top);
  hipLaunchKernelGGL(k_scale<T>, dim3((unsigned)(1 + (clear < 512 ? clear : 512))), dim3(1024), 0, s, a->g, v.total, a->rows, a->reduction, (const float*)f.top, f.tops, scale,
                     a->target, a->ignore_index, a->k, (T*)a->dx);
  const Staging sx = staging<T>(a->x, a->ldx, a->rows, a->k, f.x, true, v.order, live), sw = staging<T>(a->w, a->ldw, a->n, a->k, f.w);
  stage<T>(sx, sw, s);
  const Operand x = staged<T>(sx), w = staged<T>(sw);
  for (int64_t v0 = 0; v0 < a->n; v0 += f.piece) {
    const int64_t nv = a->n - v0 < f.piece ? a->n - v0 : f.piece, ld = padded<T>(nv);
    Operand wv = w;
    wv.p += v0 * w.ld;
    const Operand dz = {(const uint16_t*)f.dz, ld * NP};
    Product gz = {x, wv, a->rows, nv, up8(a->k), live, 0, 1, 0, 0};
    int rc = launch_dz<T>(gz, f.pz.size, {a->bias ? (const T*)a->bias + v0 : nullptr, a->target, v.order, v.stat, scale,
                                          a->reduction == CLID_REDUCE_NONE ? a->g : nullptr, (uint16_t*)f.dz, a->db ? (float*)f.sums : nullptr, v0, nv, ld}, s);
    if (rc != CLID_OK) return rc;
    if (a->dx) {
      const bool last = v0 + nv == a->n;
      Product g = {dz, wv, a->rows, a->k, nv, live, 0, 1, 0, 0};
      const float* before = v0 ? (const float*)f.sum : nullptr;
      if (last)
        rc = launch_out<T, false, true>(g, f.px, StoreOut<T>{nullptr, (T*)a->dx, before, scale + 1, v.order, a->k}, f.part, s);
      else
        rc = launch_out<T, false, true>(g, f.px, StoreOut<float>{nullptr, (float*)f.sum, before, nullptr, nullptr, a->k}, f.part, s);
      if (rc != CLID_OK) return rc;
    }
    if (a->dw) {
      T* to = (T*)a->dw + v0 * a->k;
      Product g = {dz, x, nv, a->k, a->rows, live, 1, 1, 0, 0};
      rc = launch_out<T, true, true>(g, f.pw, StoreOut<T>{nullptr, to, nullptr, scale + 1, nullptr, a->k}, f.part, s);
      if (rc != CLID_OK) return rc;
    }
    if (a->db) {
      const dim3 cols((unsigned)((nv + 63) / 64));
      const int per = run_rows<T>(f.pz.size);
      const float *alpha = scale + 1, *sums = (const float*)f.sums;
      if (f.groups) {
        hipLaunchKernelGGL(k_colsum_join<float>, dim3(cols.x, f.groups), dim3(1024), 0, s, sums, f.runs, f.share, (int)nv, live, per, (const float*)nullptr, (float*)f.joined);
        hipLaunchKernelGGL(k_colsum_join<T>, cols, dim3(1024), 0, s, (const float*)f.joined, f.groups, f.groups, (int)nv, (const int32_t*)nullptr, 1, alpha, (T*)a->db + v0);
      } else {
        hipLaunchKernelGGL(k_colsum_join<T>, cols, dim3(1024), 0, s, sums, f.runs, f.runs, (int)nv, live, per, alpha, (T*)a->db + v0);
      }
    }
  }
  return CLID_OK;
}

bool label_ok(const clid_label_args* a) { return a && sizes_ok(a->rows, a->k, a->n) && dtype_ok(a->dtype); }

template <typename T>
struct Label {
  Plan p;
  int strips;
  char *x, *w, *part, *at;
  int64_t bytes;
  explicit Label(const clid_label_args* a) {
    Ws ws(a->ws);
    p = plan<Kind<T>::NP>(a->rows, a->n, a->k, false);
    strips = (a->n + strip_width<T>(p.size) - 1) / strip_width<T>(p.size);
    x = ws.take(stage_bytes<T>(a->x, a->ldx, a->rows, a->k));
    w = ws.take(stage_bytes<T>(a->w, a->ldw, a->n, a->k));
    part = ws.take((int64_t)strips * a->rows * 8);
    at = ws.take((int64_t)strips * a->rows * 4);
    bytes = ws.used;
  }
};
template <typename T>
int label(const clid_label_args* a, hipStream_t s) {
  const Label<T> f(a);
  const Staging x = staging<T>(a->x, a->ldx, a->rows, a->k, f.x), w = staging<T>(a->w, a->ldw, a->n, a->k, f.w);
  stage<T>(x, w, s);
  Product g = {staged<T>(x), staged<T>(w), a->rows, a->n, up8(a->k), nullptr, 0, 1, 0, 0};
  const int rc = launch_stat<T, true>(g, f.p.size, (const T*)a->bias, nullptr, nullptr, (float2*)f.part, (int32_t*)f.at, nullptr, s);
  if (rc != CLID_OK) return rc;
  const int64_t joins = (a->rows + 15) / 16;
  hipLaunchKernelGGL(k_label_join, dim3((unsigned)(joins < kMostJoins ? joins : kMostJoins)), dim3(256), 0, s, (const float2*)f.part, (const int32_t*)f.at, f.strips, a->rows, a->label, a->log_prob);
  return CLID_OK;
}

}  // namespace

extern "C" int64_t clid_ce_saved(const clid_ce_args* a) {
  if (!ce_ok(a)) return bad("clid_ce_saved", "bad argument");
  return Saved(a).bytes;
}
extern "C" int64_t clid_ce_workspace(const clid_ce_args* a) {
  if (!ce_ok(a)) return bad("clid_ce_workspace", "bad argument");
  if (is_narrow(a->k, a->n) && a->rows) return narrow_ce_bytes(a);
  if (is_few(a->rows) && a->rows) return few_ce_bytes(a);
  BY_DTYPE(a->dtype, return CeFwd<T>(a).bytes;);
}
extern "C" int clid_ce_fwd(const clid_ce_args* a, void* stream) {
  const char* me = "clid_ce_fwd";
  if (!ce_ok(a)) return bad(me, "bad argument");
  if (!a->saved || (uintptr_t)a->saved % 256 || (a->rows && (!a->x || !a->w || !a->target || a->ldx < a->k || a->ldw < a->k)) ||
      (!a->loss_out && !(a->reduction == CLID_REDUCE_NONE && a->rows == 0)))
    return bad(me, "bad pointer or row stride");
  const int64_t need = clid_ce_workspace(a);
  if (a->rows && !ws_ok(a->ws, a->ws_bytes, need)) return bad(me, "workspace too small or not aligned to 256 bytes");
  int rc = CLID_OK;
  if (is_narrow(a->k, a->n) && a->rows) rc = narrow_ce(a, (hipStream_t)stream);
  else if (is_few(a->rows) && a->rows) rc = few_ce(a, Saved(a).stat, Saved(a).total, (hipStream_t)stream);
  else BY_DTYPE(a->dtype, rc = ce_fwd<T>(a, (hipStream_t)stream););
  if (rc != CLID_OK) return rc;
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}
extern "C" int64_t clid_ce_bwd_workspace(const clid_ce_args* a) {
  if (!ce_ok(a)) return bad("clid_ce_bwd_workspace", "bad argument");
  if (is_narrow(a->k, a->n)) return narrow_ce_bwd_bytes(a);
  if (is_few(a->rows)) return few_ce_bwd_bytes(a);
  BY_DTYPE(a->dtype, return CeBwd<T>(a).bytes;);
}
extern "C" int clid_ce_bwd(const clid_ce_args* a, void* stream) {
  const char* me = "clid_ce_bwd";
  if (!ce_ok(a)) return bad(me, "bad argument");
  if (a->rows == 0) return bad(me, "no rows");
  if (!a->x || !a->w || !a->target || !a->saved || (uintptr_t)a->saved % 256 || !a->g || a->ldx < a->k || a->ldw < a->k) return bad(me, "bad pointer or row stride");
  const int64_t need = clid_ce_bwd_workspace(a);
  if (!ws_ok(a->ws, a->ws_bytes, need)) return bad(me, "workspace too small or not aligned to 256 bytes");
  int rc = CLID_OK;
  if (is_narrow(a->k, a->n)) rc = narrow_ce_bwd(a, (hipStream_t)stream);
  else if (is_few(a->rows)) rc = few_ce_bwd(a, Saved(a).stat, Saved(a).total, (hipStream_t)stream);
  else BY_DTYPE(a->dtype, rc = ce_bwd<T>(a, (hipStream_t)stream););
  if (rc != CLID_OK) return rc;
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}

extern "C" int64_t clid_label_workspace(const clid_label_args* a) {
  if (!label_ok(a)) return bad("clid_label_workspace", "bad argument");
  if (is_narrow(a->k, a->n)) return 0;
  if (is_few(a->rows)) return few_label_bytes(a);
  BY_DTYPE(a->dtype, return Label<T>(a).bytes;);
}
extern "C" int clid_label_fwd(const clid_label_args* a, void* stream) {
  const char* me = "clid_label_fwd";
  if (!label_ok(a)) return bad(me, "bad argument");
  if (a->rows == 0) return CLID_OK;
  if (!a->x || !a->w || !a->label || !a->log_prob || a->ldx < a->k || a->ldw < a->k) return bad(me, "bad pointer or row stride");
  const int64_t need = clid_label_workspace(a);
  if (!ws_ok(a->ws, a->ws_bytes, need)) return bad(me, "workspace too small or not aligned to 256 bytes");
  int rc = CLID_OK;
  if (is_narrow(a->k, a->n)) rc = narrow_label(a, (hipStream_t)stream);
  else if (is_few(a->rows)) rc = few_label(a, (hipStream_t)stream);
  else BY_DTYPE(a->dtype, rc = label<T>(a, (hipStream_t)stream););
  if (rc != CLID_OK) return rc;
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}
