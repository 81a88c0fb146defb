// The dense operators for a few rows (decoding single points or tokens): at most 32 rows of x, so a layer or a class head costs its weight's
// bytes and nothing else.
//
// w goes from memory to the matrix instruction's registers directly: lane l of a wave holds 16 bytes of row l % 16 of a tile, 4 lanes 64
// neighbouring bytes of it, and the same of x as the column operand (32 k of 16 bits: 16 x 16 x 32; 16 k of fp32: four 16 x 16 x 4, exact
// fp32).  No LDS in the loop, four steps of loads in flight.  A block's waves share the tile's k; their sums meet in LDS in their order.
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
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
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
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma16(fw[u][i], fx[u][j], acc[i][j]);
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
      for (int j = 0; j < MT; ++j) acc[i][j] = mfma16(fw[i], fx[j], acc[i][j]);
  }
  // lane: column m = lane % 16, rows 4 (lane / 16) ..
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) lds[(j * 16 * NT + i * 16 + 4 * (lane >> 4) + r) * kFewRow + row] = acc[i][j][r];
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

// part[block][m]: running statistics of the block's columns
template <typename T, int MT, int NT>
__global__ void __launch_bounds__(256) k_few_label(Few a, const T* bias, Stat* part) {
  extern __shared__ __align__(16) char lds[];
  constexpr int kTile = MT * NT * 16 * kFewRow, kEach = 16 / MT;  // 256 threads: 16 MT rows, kEach threads each
  float* sums = (float*)lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int from, to;
  few_share<T>(a, wave, 4, &from, &to);
  const int m = threadIdx.x / kEach, sub = threadIdx.x % kEach;
  Stat s = {neg_inf(), 0.f, 0x7fffffff};
  const int64_t tiles = (a.n + 16 * NT - 1) / (16 * NT);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    few_tile<T, MT, NT>(a, tile * 16 * NT, from, to, threadIdx.x & 63, sums + wave * kTile);
    __syncthreads();
    if (m < a.m)
      for (int n = sub; n < 16 * NT; n += kEach) {
        const int64_t col = tile * 16 * NT + n;
        if (col >= a.n) break;
        const int at = ((m >> 4) * 16 * NT + n) * kFewRow + (m & 15);
        const float z = sums[at] + sums[kTile + at] + sums[2 * kTile + at] + sums[3 * kTile + at] + (bias ? up(bias[col]) : 0.f);
        s = join(s, {z, z != z ? z : 0.f, (int)col});
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
    const LinearOut<T> o = {(const T*)a->bias, (const T*)a->residual, (T*)a->y, (T*)a->z_out, a->ldr, a->n, a->act};
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

static int few_label_blocks(int64_t n) {
  const int64_t tiles = (n + 63) / 64;
  return (int)(tiles < 4 * kCus ? tiles : 4 * kCus);
}
int64_t few_label_bytes(const clid_label_args* a) { return up256((int64_t)few_label_blocks(a->n) * a->rows * (int64_t)sizeof(Stat)); }
int few_label(const clid_label_args* a, hipStream_t s) {
  const int blocks = few_label_blocks(a->n);
  BY_DTYPE(a->dtype, {
    const Few f = {a->x, a->w, a->ldx, a->ldw, (int)a->rows, a->k, a->n};
    Stat* part = (Stat*)a->ws;
    if (a->rows <= 16) hipLaunchKernelGGL((k_few_label<T, 1, 4>), dim3(blocks), dim3(256), 4 * 64 * kFewRow * 4, s, f, (const T*)a->bias, part);
    else hipLaunchKernelGGL((k_few_label<T, 2, 4>), dim3(blocks), dim3(256), 8 * 64 * kFewRow * 4, s, f, (const T*)a->bias, part);
    hipLaunchKernelGGL(k_few_label_join, dim3((unsigned)a->rows), dim3(256), 0, s, (const Stat*)part, blocks, (int)a->rows, a->label, a->log_prob);
    return CLID_OK;
  });
}

}  // namespace clid_dense
