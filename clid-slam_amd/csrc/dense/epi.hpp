// What the tiles' sums become: a layer's output, a gradient, a row's softmax statistics, a piece of dz.
// Each is called with one lane's 16 TN sums of a row m: element (i, r) is column nw + 32 i + 8 (r / 4) + 4 half + r % 4.
#pragma once
#include "tile.hpp"

namespace clid_dense {

template <typename T> struct Four;  // four neighbouring values of a type as one load or store
template <> struct Four<float> { using V = float4; };
template <> struct Four<bf16> { using V = ushort4; };
template <> struct Four<f16> { using V = ushort4; };

template <typename T>
__device__ __forceinline__ void put4(T* p, const float (&v)[4], int count, bool wide) {
  if (wide && count >= 4) {
    union { typename Four<T>::V w; T t[4]; } u;
#pragma unroll
    for (int q = 0; q < 4; ++q) u.t[q] = down<T>(v[q]);
    *(typename Four<T>::V*)p = u.w;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < count) p[q] = down<T>(v[q]);
  }
}
template <typename T>
__device__ __forceinline__ void get4(const T* p, float (&v)[4], int count, bool wide) {
  if (wide && count >= 4) {
    union { typename Four<T>::V w; T t[4]; } u;
    u.w = *(const typename Four<T>::V*)p;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = up(u.t[q]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = q < count ? up(p[q]) : 0.f;
  }
}

// z + bias -> act -> + residual -> y, and z for the backward pass; also behind a sum over splits (k_join)
template <typename T>
struct LinearOut {
  const T *bias, *res;
  T *y, *z;
  int64_t ldr, n;
  int act, wide, res_wide;  // 4 neighbouring values of y and z (of res) are one aligned store (load)
  // (v: four sums at row m, column c)
  __device__ __forceinline__ void four(float (&v)[4], const float (&b)[4], int64_t m, int64_t c) const {
    const int count = (int)(n - c < 4 ? n - c : 4);
    if (count <= 0) return;
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (res) get4(res + m * ldr + c, r, count, res_wide);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += b[q];
    if (z) {
      if (wide && count >= 4) {
        union { typename Four<T>::V w; T t[4]; } u;
#pragma unroll
        for (int q = 0; q < 4; ++q) u.t[q] = keep_z<T>(v[q]);
        *(typename Four<T>::V*)(z + m * n + c) = u.w;
      } else {
        for (int q = 0; q < count; ++q) z[m * n + c + q] = keep_z<T>(v[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = act_value(v[q], act) + r[q];
    put4(y + m * n + c, v, count, wide);
  }
};

// bias of the tile's columns in LDS as fp32
template <typename T>
__device__ __forceinline__ void stage_bias(const T* bias, int64_t n0, int64_t n, int cols, char* lds) {
  for (int c = threadIdx.x; c < cols; c += blockDim.x) ((float*)lds)[c] = bias && n0 + c < n ? up(bias[n0 + c]) : 0.f;
}

template <typename T, int BN>
struct EpiLinear {
  LinearOut<T> o;
  __device__ __forceinline__ void prepare(int64_t n0, char* lds) const { stage_bias(o.bias, n0, o.n, BN, lds); }
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t m, bool on, int64_t nw, int64_t n, int half, int, const char* lds, int at) const {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * i + 8 * j + 4 * half;
        const float4 b4 = *(const float4*)(lds + (at + c) * 4);
        float v[4] = {acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]};
        const float b[4] = {b4.x, b4.y, b4.z, b4.w};
        o.four(v, b, m, nw + c);
      }
  }
};

// out[order ? order[m] : m] = alpha sum + add
template <typename T>
struct StoreOut {
  T* out;
  const float *add, *alpha;  // add: [m][n] fp32 of the pieces before
  const int32_t* order;
  int64_t n;
  int wide;
  __device__ __forceinline__ void four(float (&v)[4], const float (&)[4], int64_t m, int64_t c) const {
    const int count = (int)(n - c < 4 ? n - c : 4);
    if (count <= 0) return;
    if (add) {
      float a[4];
      get4(add + m * n + c, a, count, n % 4 == 0);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += a[q];
    }
    const float s = alpha ? *alpha : 1.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] *= s;
    put4(out + (order ? (int64_t)order[m] : m) * n + c, v, count, wide);
  }
};
template <typename T, int BN>
struct EpiStore {
  StoreOut<T> o;
  __device__ __forceinline__ void prepare(int64_t, char*) const {}
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t m, bool on, int64_t nw, int64_t, int half, int, const char*, int) const {
    if (!on) return;
    const float b[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v[4] = {acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]};
        o.four(v, b, m, nw + 32 * i + 8 * j + 4 * half);
      }
  }
};

// part[split][m][n4] = sum over this block's share of k (n4: n up to 4)
template <int BN>
struct EpiPart {
  float* part;
  int64_t m, n4;
  __device__ __forceinline__ void prepare(int64_t, char*) const {}
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t mm, bool on, int64_t nw, int64_t, int half, int split, const char*, int) const {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t c = nw + 32 * i + 8 * j + 4 * half;
        if (c < n4) *(float4*)(part + ((int64_t)split * m + mm) * n4 + c) = float4{acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]};
      }
  }
};

// the splits' sums joined in their order, four columns a thread, and handed on
template <typename T, class Out>
__global__ void __launch_bounds__(256) k_join(const float* part, int splits, int64_t m, int64_t n4, const int32_t* live, const T* bias, Out o) {
  const int64_t rows = live && *live < m ? *live : m;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * (n4 / 4); i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / (n4 / 4), c = (i - r * (n4 / 4)) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float4 p = *(const float4*)(part + ((int64_t)s * m + r) * n4 + c);
      v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
    }
    if (bias)
      for (int q = 0; q < 4; ++q) b[q] = c + q < o.n ? up(bias[c + q]) : 0.f;
    o.four(v, b, r, c);
  }
}

// softmax statistics of this wave's 32 TN columns for each of its rows -> part[strip][m] (m, r), at: the column of m where labels are
// asked; the target's z -> zt[m]
template <typename T, int BN, int STRIP, bool LABEL>
struct EpiStat {
  const T* bias;
  const int64_t* target;  // with order: the row's target is target[order[m]]
  const int32_t* order;
  float2* part;
  int32_t* part_at;
  float* zt;
  int64_t m_all, n;
  __device__ __forceinline__ void prepare(int64_t n0, char* lds) const { stage_bias(bias, n0, n, BN, lds); }
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t m, bool on, int64_t nw, int64_t, int half, int, const char* lds, int at) const {
    if (nw >= n) return;
    int t = -1;
    if constexpr (!LABEL) {
      if (on) {
        const int64_t tt = target[order[m]];
        t = tt >= nw && tt < nw + 32 * TN ? (int)(tt - nw) : -1;
      }
    }
    float top = neg_inf();
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * i + 8 * j + 4 * half;
        const float4 b4 = *(const float4*)(lds + (at + c) * 4);
        const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float z = acc[i][4 * j + q] + b[q];
          if constexpr (!LABEL)
            if (t == c + q) zt[m] = z;
          z = nw + c + q < n ? z : neg_inf();
          acc[i][4 * j + q] = z;
          top = fmaxf(top, z);
        }
      }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float safe = top == neg_inf() ? 0.f : top;
    float rest = 0.f;
    int same = 0;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float z = acc[i][r];
        const bool is = z == top;
        rest += is ? 0.f : __builtin_amdgcn_exp2f((z - safe) * 1.4426950408889634f);
        same += is;
      }
    rest += __shfl_xor(rest, 32, 64);
    same += __shfl_xor(same, 32, 64);
    // columns that share the largest value: one of them is `m`, the others count as exp(0); without a finite value none does
    rest = top == neg_inf() ? (rest == rest ? 0.f : rest) : rest + (float)(same - 1);
    if (top == __builtin_inff()) rest = __builtin_nanf("");
    int best = 0x7fffffff;
    if constexpr (LABEL) {
      const bool odd = rest != rest;  // a NaN among the columns, or infinities
      bool nan = false;
#pragma unroll
      for (int i = TN - 1; i >= 0; --i)
#pragma unroll
        for (int r = 15; r >= 0; --r)
          if (acc[i][r] == top) best = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
      if (odd) {
        int first = 0x7fffffff;
#pragma unroll
        for (int i = TN - 1; i >= 0; --i)
#pragma unroll
          for (int r = 15; r >= 0; --r)
            if (acc[i][r] != acc[i][r]) first = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
        const int other = __shfl_xor(first, 32, 64);
        first = other < first ? other : first;
        nan = first != 0x7fffffff;
        if (nan) best = first;
      }
      if (nan) top = __builtin_nanf("");
      const int other = __shfl_xor(best, 32, 64);
      best = other < best ? other : best;
    }
    if (half == 0 && on) {
      const int64_t strip = nw / STRIP;
      part[strip * m_all + m] = float2{top, rest};
      if constexpr (LABEL) part_at[strip * m_all + m] = (int)nw + best;
    }
  }
};

// dz of a piece of the classes, in NP planes: (p - onehot) x the row's factor
template <typename T, int BN, int NP>
struct EpiDz {
  const T* bias;  // of the piece
  const int64_t* target;
  const int32_t* order;
  const float4* stat;  // [row in order]
  const float* scale;  // [0]: what every row is multiplied by
  const float* g;      // per-row factor, by original row, or NULL
  uint16_t* dz;
  int64_t v0, n, ld, plane;  // columns v0 .. v0 + n, ld: n up to 8 (zeros there)
  __device__ __forceinline__ void prepare(int64_t n0, char* lds) const { stage_bias(bias, n0, n, BN, lds); }
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t m, bool on, int64_t nw, int64_t, int half, int, const char* lds, int at) const {
    if (!on) return;
    const int64_t from = order[m];
    const float4 s = stat[m];
    const int64_t tt = target[from] - v0 - nw;
    const int t = tt >= 0 && tt < 32 * TN ? (int)tt : -1;
    float f = scale[0];
    if (g) f *= g[from];
    const float inv = s.w != s.w ? s.w : s.y * f, hit = s.z * f;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * i + 8 * j + 4 * half;
        if (nw + c >= ld) continue;
        const float4 b4 = *(const float4*)(lds + (at + c) * 4);
        const float b[4] = {b4.x, b4.y, b4.z, b4.w};
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float p = __builtin_amdgcn_exp2f((acc[i][4 * j + q] + b[q] - s.x) * 1.4426950408889634f) * inv;
          v[q] = nw + c + q < n ? (t == c + q ? hit : p) : 0.f;
        }
        uint16_t* to = dz + m * ld + nw + c;
        if constexpr (NP == 1) {
          union { ushort4 w; T t[4]; } u;
#pragma unroll
          for (int q = 0; q < 4; ++q) u.t[q] = down<T>(v[q]);
          *(ushort4*)to = u.w;
        } else {
          union { ushort4 w; uint16_t t[4]; } u[3];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint16_t h[3];
            planes(v[q], h);
            for (int s3 = 0; s3 < 3; ++s3) u[s3].t[q] = h[s3];
          }
#pragma unroll
          for (int s3 = 0; s3 < 3; ++s3) *(ushort4*)(to + s3 * plane) = u[s3].w;
        }
      }
  }
};

}  // namespace clid_dense
