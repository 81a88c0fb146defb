// The dense operators for a few rows (decoding single points or tokens): at most 32 rows of x, so a layer or a class head costs its weight's
// bytes and nothing else.
//
// w goes from memory to the matrix instruction's registers directly: lane l of a wave holds 16 bytes of row l % 16 of a tile, 4 lanes 64
// neighbouring bytes of it, and the same of x as the column operand (32 k of 16 bits: 16 x 16 x 32; 16 k of fp32: four 16 x 16 x 4, exact
// fp32).  No LDS in the loop, four steps of loads in flight.  A block's waves share the tile's k; their sums meet in LDS in their order.
// The cross entropy's backward pass makes z again the same way, leaves dz in fp32 (32 rows of it are small) and takes both products on the fp32
// matrix instruction (16 x 16 x 4), w and dw in 16 bytes a lane of 256 neighbouring ones: with few rows nothing averages a rounding of
// dz away, and the products cost nothing beside the weight's bytes.
// Bound by the weight's bytes: 1 x 4096 -> 8192 bf16 silu 13.5 us, label of 1 x 4096 -> 131072 bf16 215 us, both 5.0 TB/s (a large copy: 4.8).
// Where n is large a wave takes 4 tiles at once (one read of x for four of w) and a block goes through many, keeping running softmax
// statistics, so that a head of 131072 classes leaves one partial result per block.
#include "stage.hpp"

namespace clid_dense {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

struct Few {
  const void *x, *w;
  int64_t ldx, ldw;
  int m, k;
  int64_t n;
};

template <typename T> struct Frag {  // 16 bytes of a row
  static constexpr int kElems = 16 / sizeof(T), kStep = 4 * kElems;
  T t[kElems];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(t, p, 16); }  // rows need no alignment
  __device__ __forceinline__ void load(const T* p, int count) {
#pragma unroll
    for (int e = 0; e < kElems; ++e) t[e] = e < count ? p[e] : down<T>(0.f);
  }
};
__device__ __forceinline__ f32x4 mfma16(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(const Frag<f16>& a, const Frag<f16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.t[e], b.t[e], c, 0, 0, 0);
  return c;
}

constexpr int kFewRow = 17;  // floats between a tile's rows in LDS

// sums of rows n0 .. n0 + 16 NT of w with the rows of x, over this wave's share of k -> lds[n][m]
template <typename T, int MT, int NT>
__device__ __forceinline__ void few_tile(const Few& a, int64_t n0, int k_from, int k_to, int lane, float* lds) {
  using F = Frag<T>;
  const int row = lane & 15, kk = (lane >> 4) * F::kElems;
  const T *x[MT], *w[NT];
#pragma unroll
  for (int j = 0; j < MT; ++j) x[j] = (const T*)a.x + (j * 16 + row < a.m ? j * 16 + row : a.m - 1) * a.ldx + kk;  // rows that are not there: the last one's
#pragma unroll
  for (int i = 0; i < NT; ++i) w[i] = (const T*)a.w + (n0 + i * 16 + row < a.n ? n0 + i * 16 + row : a.n - 1) * a.ldw + kk;
  f32x4 acc[2][NT][MT];  // every other step's: half as many roundings in a row
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[0][i][j] = acc[1][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int k = k_from;
  constexpr int kDeep = NT == 1 ? 8 : 4;
  for (; k + kDeep * F::kStep <= k_to; k += kDeep * F::kStep) {
    F fw[kDeep][NT], fx[kDeep][MT];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
#pragma unroll
      for (int i = 0; i < NT; ++i) fw[u][i].load(w[i] + k + u * F::kStep);
#pragma unroll
      for (int j = 0; j < MT; ++j) fx[u][j].load(x[j] + k + u * F::kStep);
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[u & 1][i][j] = mfma16(fw[u][i], fx[u][j], acc[u & 1][i][j]);
  }
  for (; k < k_to; k += F::kStep) {
    F fw[NT], fx[MT];
    const int left = k_to - k - kk, count = left > F::kElems ? F::kElems : left;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (k + F::kStep <= k_to) fw[i].load(w[i] + k);
      else fw[i].load(w[i] + k, count);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      if (k + F::kStep <= k_to) fx[j].load(x[j] + k);
      else fx[j].load(x[j] + k, count);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[0][i][j] = mfma16(fw[i], fx[j], acc[0][i][j]);
  }
  // lane: column m = lane % 16, rows 4 (lane / 16) ..
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) lds[(j * 16 * NT + i * 16 + 4 * (lane >> 4) + r) * kFewRow + row] = acc[0][i][j][r] + acc[1][i][j][r];
}
// wave's share of k, in whole steps
template <typename T>
__device__ __forceinline__ void few_share(const Few& a, int wave, int waves, int* from, int* to) {
  const int steps = (a.k + Frag<T>::kStep - 1) / Frag<T>::kStep, per = (steps + waves - 1) / waves * Frag<T>::kStep;
  *from = wave * per < a.k ? wave * per : a.k;
  *to = *from + per < a.k ? *from + per : a.k;
}

template <typename T, int MT, int NT>
__global__ void __launch_bounds__(NT == 1 ? 1024 : 256) k_few_linear(Few a, LinearOut<T> o) {
  extern __shared__ __align__(16) char lds[];
  constexpr int kTile = MT * NT * 16 * kFewRow;
  float* sums = (float*)lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  int from, to;
  few_share<T>(a, wave, waves, &from, &to);
  const int64_t tile = blockIdx.x;
  few_tile<T, MT, NT>(a, tile * 16 * NT, from, to, threadIdx.x & 63, sums + wave * kTile);
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 16 * 16 * NT; e += blockDim.x) {
    const int n = e % (16 * NT), m = e / (16 * NT);
    const int64_t col = tile * 16 * NT + n;
    if (m >= a.m || col >= a.n) continue;
    float v = 0.f;
    for (int i = 0; i < waves; ++i) v += sums[i * kTile + ((m >> 4) * 16 * NT + n) * kFewRow + (m & 15)];
    o.one(v, m, col);
  }
}

// part[block][m]: running statistics of the block's columns; zt[m]: the target's z, where there are targets
template <typename T, int MT, int NT>
__global__ void __launch_bounds__(256) k_few_stat(Few a, const T* bias, const int64_t* target, float* zt, Stat* part) {
  extern __shared__ __align__(16) char lds[];
  constexpr int kTile = MT * NT * 16 * kFewRow, kEach = 16 / MT;  // 256 threads: 16 MT rows, kEach threads each
  float* sums = (float*)lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int from, to;
  few_share<T>(a, wave, 4, &from, &to);
  const int m = threadIdx.x / kEach, sub = threadIdx.x % kEach;
  Stat s = {neg_inf(), 0.f, 0x7fffffff};
  const int64_t tiles = (a.n + 16 * NT - 1) / (16 * NT), t = target && m < a.m ? target[m] : -1;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    few_tile<T, MT, NT>(a, tile * 16 * NT, from, to, threadIdx.x & 63, sums + wave * kTile);
    __syncthreads();
    if (m < a.m)
      for (int n = sub; n < 16 * NT; n += kEach) {
        const int64_t col = tile * 16 * NT + n;
        if (col >= a.n) break;
        const int at = ((m >> 4) * 16 * NT + n) * kFewRow + (m & 15);
        const float z = sums[at] + sums[kTile + at] + sums[2 * kTile + at] + sums[3 * kTile + at] + (bias ? up(bias[col]) : 0.f);
        s = join(s, {z, z < __builtin_inff() ? 0.f : __builtin_nanf(""), (int)col});  // (+inf - inf or a NaN: no sum is a number)
        if (t == col) zt[m] = z;
      }
    __syncthreads();
  }
#pragma unroll
  for (int d = 1; d < kEach; d <<= 1) s = join(s, {__shfl_xor(s.m, d, 64), __shfl_xor(s.r, d, 64), __shfl_xor(s.at, d, 64)});
  if (sub == 0 && m < a.m) part[(int64_t)blockIdx.x * a.m + m] = s;
}
// a block a row
__global__ void __launch_bounds__(256) k_few_label_join(const Stat* part, int blocks, int rows, int64_t* label, float* log_prob) {
  __shared__ Stat p[4];
  Stat s = {neg_inf(), 0.f, 0x7fffffff};
  for (int b = threadIdx.x; b < blocks; b += 256) s = join(s, part[(int64_t)b * rows + blockIdx.x]);
  for (int d = 1; d < 64; d <<= 1) s = join(s, {__shfl_xor(s.m, d, 64), __shfl_xor(s.r, d, 64), __shfl_xor(s.at, d, 64)});
  if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = join(join(p[0], p[1]), join(p[2], p[3]));
  label[blockIdx.x] = s.at;
  log_prob[blockIdx.x] = s.m == neg_inf() ? __builtin_nanf("") : -log1pf(s.r);
}

template <typename T, int MT, int NT>
static int few_linear_launch(const Few& f, const LinearOut<T>& o, int waves, hipStream_t s) {
  const int lds = waves * MT * NT * 16 * kFewRow * 4;
  const int rc = allow_lds((const void*)k_few_linear<T, MT, NT>, lds);
  if (rc != CLID_OK) return rc;
  hipLaunchKernelGGL((k_few_linear<T, MT, NT>), dim3((unsigned)((f.n + 16 * NT - 1) / (16 * NT))), dim3(64 * waves), lds, s, f, o);
  return CLID_OK;
}
int few_linear(const clid_linear_args* a, hipStream_t s) {
  BY_DTYPE(a->dtype, {
    const Few f = {a->x, a->w, a->ldx, a->ldw, (int)a->rows, a->k, a->n};
    const LinearOut<T> o = {(const T*)a->bias, (const T*)a->residual, (T*)a->y, (KeptZ<T>::Z*)a->z_out, a->ldr, a->n, a->act};
    const int steps = (a->k + Frag<T>::kStep - 1) / Frag<T>::kStep;
    if (a->n >= 64 * 1024) {  // 1024 blocks of 64 columns
      const int waves = steps >= 16 ? 4 : steps >= 8 ? 2 : 1;
      return a->rows <= 16 ? few_linear_launch<T, 1, 4>(f, o, waves, s) : few_linear_launch<T, 2, 4>(f, o, waves, s);
    }
    int waves = 1;
    while (waves < 16 && steps >= 16 * waves) waves *= 2;  // at least 8 steps a wave
    return a->rows <= 16 ? few_linear_launch<T, 1, 1>(f, o, waves, s) : few_linear_launch<T, 2, 1>(f, o, waves, s);
  });
}

static int few_blocks(int64_t n) {
  const int64_t tiles = (n + 63) / 64;
  return (int)(tiles < 4 * kCus ? tiles : 4 * kCus);
}
int64_t few_label_bytes(const clid_label_args* a) { return up256((int64_t)few_blocks(a->n) * a->rows * (int64_t)sizeof(Stat)); }
int few_label(const clid_label_args* a, hipStream_t s) {
  const int blocks = few_blocks(a->n);
  BY_DTYPE(a->dtype, {
    const Few f = {a->x, a->w, a->ldx, a->ldw, (int)a->rows, a->k, a->n};
    Stat* part = (Stat*)a->ws;
    if (a->rows <= 16) hipLaunchKernelGGL((k_few_stat<T, 1, 4>), dim3(blocks), dim3(256), 4 * 64 * kFewRow * 4, s, f, (const T*)a->bias, (const int64_t*)nullptr, (float*)nullptr, part);
    else hipLaunchKernelGGL((k_few_stat<T, 2, 4>), dim3(blocks), dim3(256), 8 * 64 * kFewRow * 4, s, f, (const T*)a->bias, (const int64_t*)nullptr, (float*)nullptr, part);
    hipLaunchKernelGGL(k_few_label_join, dim3((unsigned)a->rows), dim3(256), 0, s, (const Stat*)part, blocks, (int)a->rows, a->label, a->log_prob);
    return CLID_OK;
  });
}


// ---- cross entropy ----------------------------------------------------------------------------------------------------------

// a row's statistics joined (32 threads a row), its loss, and the sums: one block
__global__ void __launch_bounds__(1024) k_few_loss(const Stat* part, int blocks, const float* zt, const int64_t* target, int rows, int n, int64_t ignore,
                                                   int reduction, float4* stat, float* total, float* loss_out) {
  __shared__ double sums[32];
  __shared__ int counts[32];
  const int m = threadIdx.x >> 5, sub = threadIdx.x & 31;
  Stat s = {neg_inf(), 0.f, 0x7fffffff};
  if (m < rows)
#pragma unroll 4
    for (int b = sub; b < blocks; b += 32) s = join(s, part[(int64_t)b * rows + m]);
  for (int d = 1; d < 32; d <<= 1) s = join(s, {__shfl_xor(s.m, d, 64), __shfl_xor(s.r, d, 64), __shfl_xor(s.at, d, 64)});
  if (sub == 0) {
    double l = 0.0;
    int c = 0;
    if (m < rows) {
      const int64_t t = target[m];
      float loss = 0.f;
      if (t != ignore) {
        loss = t >= 0 && t < n ? (s.m - zt[m]) + log1pf(s.r) : __builtin_nanf("");
        c = 1;
      }
      stat[m] = {s.m, 1.f / (1.f + s.r), expm1f(-loss), loss};
      if (reduction == CLID_REDUCE_NONE) loss_out[m] = loss;
      l = loss;
    }
    sums[m] = l;
    counts[m] = c;
  }
  __syncthreads();
  if (threadIdx.x) return;
  double l = 0.0;
  int c = 0;
  for (int i = 0; i < 32; ++i) {
    l += sums[i];
    c += counts[i];
  }
  total[0] = (float)l;
  total[1] = (float)c;
  if (reduction == CLID_REDUCE_MEAN) loss_out[0] = c ? (float)(l / c) : 0.f;
  if (reduction == CLID_REDUCE_SUM) loss_out[0] = (float)l;
}

// dz[m][np] in fp32 (zeros behind n, and in rows that do not count or are not there up to 16 MT), db
template <typename T, int MT, int NT>
__global__ void __launch_bounds__(256) k_few_dz(Few a, const T* bias, const int64_t* target, int64_t ignore, const float4* stat, const float* g, int reduction,
                                                const float* total, float* dz, int64_t np, T* db) {
  extern __shared__ __align__(16) char lds[];
  constexpr int kTile = MT * NT * 16 * kFewRow, kCols = 16 * NT, kGroups = 256 / kCols;
  float* sums = (float*)lds;
  __shared__ float sb[kGroups][kCols];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int from, to;
  few_share<T>(a, wave, 4, &from, &to);
  const int64_t n0 = (int64_t)blockIdx.x * kCols;
  few_tile<T, MT, NT>(a, n0, from, to, threadIdx.x & 63, sums + wave * kTile);
  __syncthreads();
  const int n = threadIdx.x % kCols, group = threadIdx.x / kCols;
  const int64_t col = n0 + n;
  const float b = bias && col < a.n ? up(bias[col]) : 0.f;
  float all = 0.f;
  for (int m = group; m < 16 * MT; m += kGroups) {
    float v = 0.f;
    if (m < a.m && col < a.n && target[m] != ignore) {
      const float4 s = stat[m];
      const int at = ((m >> 4) * kCols + n) * kFewRow + (m & 15);
      const float z = sums[at] + sums[kTile + at] + sums[2 * kTile + at] + sums[3 * kTile + at] + b;
      const float f = reduction == CLID_REDUCE_NONE ? g[m] : reduction == CLID_REDUCE_MEAN ? g[0] / fmaxf(total[1], 1.f) : g[0];
      v = f * (s.w != s.w ? s.w : target[m] == col ? s.z : __builtin_amdgcn_exp2f((z - s.x) * 1.4426950408889634f) * s.y);
    }
    dz[m * np + col] = v;
    all += v;
  }
  sb[group][n] = all;
  __syncthreads();
  if (db && group == 0 && col < a.n) {
    for (int i = 1; i < kGroups; ++i) all += sb[i][n];
    db[col] = down<T>(all);
  }
}

// a layer's: dz = dy act'(z)
template <int MT>
__global__ void __launch_bounds__(256) k_few_linear_dz(const float* dy, int64_t lddy, const float* z, int rows, int64_t n, int act, float* dz, int64_t np, float* db) {
  __shared__ float sums[4][64];
  const int c = threadIdx.x & 63, group = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  float all = 0.f;
#pragma unroll
  for (int m = group; m < 16 * MT; m += 4) {
    float v = 0.f;
    if (m < rows && col < n) {
      v = dy[m * lddy + col];
      if (z) v = act_grad(v, z[m * n + col], act);
    }
    dz[m * np + col] = v;
    all += v;
  }
  sums[group][c] = all;
  __syncthreads();
  if (db && group == 0 && col < n) db[col] = all + sums[1][c] + sums[2][c] + sums[3][c];
}

// dx: block (128 columns of k, share of n) -> part[share][16 MT][k up to 128].  Lane l: 8 neighbouring columns 8 (l % 16) of row 4 (l / 16) + c of 16
// rows of w, c = 0 .. 3; instruction j takes column j of the eight.
template <typename T, int MT>
__global__ void __launch_bounds__(256) k_few_dx(Few a, const float* dz, int64_t np, int64_t per, float* part) {
  __shared__ float sums[3][MT * 16][128 + 4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const int k0 = blockIdx.x * 128 + 8 * i, count = a.k - k0;
  const int64_t v_end = (blockIdx.y + 1) * per < np ? (blockIdx.y + 1) * per : np;
  f32x4 acc[MT][8];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int64_t v = blockIdx.y * per + wave * 16; v < v_end; v += 64) {  // np is a multiple of 64
    float w[4][8], d[MT][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t row = v + 4 * q + c;
      get8((const T*)a.w + row * a.ldw + k0, w[c], row < a.n ? count : 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) *(float4*)d[t] = *(const float4*)(dz + (t * 16 + i) * np + v + 4 * q);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(d[t][c], w[c][j], acc[t][j], 0, 0, 0);
  }
  // lane: rows 4 q + r, columns 8 i + j
  if (wave)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[wave - 1][t * 16 + 4 * q + r][8 * i + j] = acc[t][j][r];
  __syncthreads();
  if (wave) return;
  const int64_t kp = (int64_t)gridDim.x * 128;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = t * 16 + 4 * q + r;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = acc[t][j][r] + sums[0][m][8 * i + j] + sums[1][m][8 * i + j] + sums[2][m][8 * i + j];
      out8(part + (blockIdx.y * (int64_t)(16 * MT) + m) * kp + k0, v, 8);
    }
}
template <typename T>
__global__ void __launch_bounds__(256) k_few_dx_join(const float* part, int shares, int rows16, int64_t kp, int rows, int k, const int64_t* target, int64_t ignore, T* dx) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)rows * k) return;
  const int m = (int)(e / k), c = (int)(e - (int64_t)m * k);
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < shares; ++i) s += part[((int64_t)i * rows16 + m) * kp + c];
  dx[e] = down<T>(target && target[m] == ignore ? 0.f : s);
}

// dw: a wave holds its 128 columns of x and walks 16 rows of dw at a time
template <typename T, int MT>
__global__ void __launch_bounds__(256) k_few_dw(Few a, const int64_t* target, int64_t ignore, const float* dz, int64_t np, T* dw) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const int k0 = blockIdx.x * 128 + 8 * i, count = a.k - k0;
  float x[4 * MT][8];
#pragma unroll
  for (int s = 0; s < 4 * MT; ++s) {
    const int m = 4 * s + q;
    const bool on = m < a.m && !(target && target[m] == ignore);  // a row that does not count is zeros whatever it holds
    get8((const T*)a.x + (int64_t)m * a.ldx + k0, x[s], on ? count : 0);
  }
  for (int64_t v = ((int64_t)blockIdx.y * 4 + wave) * 16; v < np; v += (int64_t)gridDim.y * 64) {
    float d[4 * MT];
#pragma unroll
    for (int s = 0; s < 4 * MT; ++s) d[s] = dz[(4 * s + q) * np + v + i];
    f32x4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4 * MT; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(d[s], x[s][j], acc[j], 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = v + 4 * q + r;
      T t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = down<T>(acc[j][r]);
      if (row < a.n) out8(dw + row * a.k + k0, t, count);
    }
  }
}

int64_t few_ce_bytes(const clid_ce_args* a) { return up256((int64_t)few_blocks(a->n) * a->rows * (int64_t)sizeof(Stat)) + up256(a->rows * 4); }
int few_ce(const clid_ce_args* a, float4* stat, float* total, hipStream_t s) {
  const int blocks = few_blocks(a->n);
  Stat* part = (Stat*)a->ws;
  float* zt = (float*)((char*)a->ws + up256((int64_t)blocks * a->rows * (int64_t)sizeof(Stat)));
  BY_DTYPE(a->dtype, {
    const Few f = {a->x, a->w, a->ldx, a->ldw, (int)a->rows, a->k, a->n};
    if (a->rows <= 16) hipLaunchKernelGGL((k_few_stat<T, 1, 4>), dim3(blocks), dim3(256), 4 * 64 * kFewRow * 4, s, f, (const T*)a->bias, a->target, zt, part);
    else hipLaunchKernelGGL((k_few_stat<T, 2, 4>), dim3(blocks), dim3(256), 8 * 64 * kFewRow * 4, s, f, (const T*)a->bias, a->target, zt, part);
  });
  hipLaunchKernelGGL(k_few_loss, dim3(1), dim3(1024), 0, s, (const Stat*)part, blocks, (const float*)zt, a->target, (int)a->rows, a->n, a->ignore_index,
                     a->reduction, stat, total, a->loss_out);
  return CLID_OK;
}

struct FewBwd {
  int64_t np, kp, per;
  int mt, shares;
  char *dz, *part;
  int64_t bytes;
  FewBwd(void* base, int64_t rows, int32_t k, int32_t n, bool dx) {
    Ws ws(base);
    np = ((int64_t)n + 63) / 64 * 64;
    kp = ((int64_t)k + 127) / 128 * 128;
    mt = rows <= 16 ? 1 : 2;
    // blocks of 128 columns of k and of shares of n: about 4 a CU, a share 256 rows of w at least
    int64_t want = 4 * kCus / (kp / 128), most = (np + 255) / 256;
    shares = (int)(want < 1 ? 1 : want < most ? want : most);
    per = ((np + shares - 1) / shares + 63) / 64 * 64;
    shares = (int)((np + per - 1) / per);
    dz = ws.take(16 * mt * np * 4);
    part = ws.take(dx ? (int64_t)shares * 16 * mt * kp * 4 : 0);
    bytes = ws.used;
  }
};
// dx and dw of the dz in the workspace; target NULL: every row counts
template <typename T, int MT>
static void few_products(const Few& f, const FewBwd& b, const int64_t* target, int64_t ignore, void* dx, void* dw, hipStream_t s) {
  const float* dz = (const float*)b.dz;
  const unsigned kb = (unsigned)(b.kp / 128);
  if (dx) {
    hipLaunchKernelGGL((k_few_dx<T, MT>), dim3(kb, (unsigned)b.shares), dim3(256), 0, s, f, dz, b.np, b.per, (float*)b.part);
    hipLaunchKernelGGL(k_few_dx_join<T>, dim3((unsigned)(((int64_t)f.m * f.k + 255) / 256)), dim3(256), 0, s, (const float*)b.part, b.shares, 16 * MT, b.kp, f.m, f.k, target,
                       ignore, (T*)dx);
  }
  if (dw) {
    const int64_t tiles = b.np / 64, want = 8 * kCus / kb + 1;
    hipLaunchKernelGGL((k_few_dw<T, MT>), dim3(kb, (unsigned)(tiles < want ? tiles : want)), dim3(256), 0, s, f, target, ignore, dz, b.np, (T*)dw);
  }
}

int64_t few_ce_bwd_bytes(const clid_ce_args* a) { return FewBwd(nullptr, a->rows, a->k, a->n, a->dx).bytes; }
template <typename T, int MT>
static void few_ce_bwd_launch(const clid_ce_args* a, const FewBwd& b, const float4* stat, const float* total, hipStream_t s) {
  const Few f = {a->x, a->w, a->ldx, a->ldw, (int)a->rows, a->k, a->n};
  hipLaunchKernelGGL((k_few_dz<T, MT, 4>), dim3((unsigned)(b.np / 64)), dim3(256), 4 * MT * 64 * kFewRow * 4, s, f, (const T*)a->bias, a->target, a->ignore_index, stat,
                     a->g, a->reduction, total, (float*)b.dz, b.np, (T*)a->db);
  few_products<T, MT>(f, b, a->target, a->ignore_index, a->dx, a->dw, s);
}
int few_ce_bwd(const clid_ce_args* a, const float4* stat, const float* total, hipStream_t s) {
  const FewBwd b(a->ws, a->rows, a->k, a->n, a->dx);
  BY_DTYPE(a->dtype, {
    if (b.mt == 1) few_ce_bwd_launch<T, 1>(a, b, stat, total, s);
    else few_ce_bwd_launch<T, 2>(a, b, stat, total, s);
  });
  return CLID_OK;
}

// A layer's backward pass, fp32 only: the tiles' planes of w cost more than the products (layer and gradients, gelu, 1 and 32 rows: 4096 -> 8192 in tiles
// 196 and 218 us, here 83 and 133; 1024 -> 1000: 31 and 39, 22 and 31).  16-bit operands go to the tiles as they lie (bf16 4096 -> 8192: tiles 58
// and 72 us, here 62 and 118).
int64_t few_linear_bwd_bytes(const clid_linear_bwd_args* a) { return FewBwd(nullptr, a->rows, a->k, a->n, a->dx).bytes; }
template <int MT>
static void few_linear_bwd_launch(const clid_linear_bwd_args* a, const FewBwd& b, hipStream_t s) {
  const Few f = {a->x, a->w, a->ldx, a->ldw, (int)a->rows, a->k, a->n};
  // z and y are both fp32: z_is_y makes no difference
  hipLaunchKernelGGL((k_few_linear_dz<MT>), dim3((unsigned)(b.np / 64)), dim3(256), 0, s, (const float*)a->dy, a->lddy, a->act == CLID_ACT_NONE ? nullptr : (const float*)a->z,
                     (int)a->rows, a->n, a->act, (float*)b.dz, b.np, (float*)a->db);
  few_products<float, MT>(f, b, nullptr, 0, a->dx, a->dw, s);
}
int few_linear_bwd(const clid_linear_bwd_args* a, hipStream_t s) {
  const FewBwd b(a->ws, a->rows, a->k, a->n, a->dx);
  if (b.mt == 1) few_linear_bwd_launch<1>(a, b, s);
  else few_linear_bwd_launch<2>(a, b, s);
  return CLID_OK;
}

}  // namespace clid_dense
