// What the tiles' sums become: a layer's output, a gradient, a row's softmax statistics, a piece of dz.
// Each gets a wave's sums: of 32 rows, lane l holds row m_first + l % 32, its element (i, r) column nw + 32 i + 8 (r / 4) + 4 (l / 32) + r % 4.
#pragma once
#include "tile.hpp"

namespace clid_dense {

// 8 neighbouring values of a row, by 16 bytes (which need no more alignment than the values) where there are 8
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ void get8(const T* p, float (&v)[8], int count) {
  if (count >= 8) {
    union { words4 w[sizeof(T) / 2]; T t[8]; } u;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.w[i] = ((const words4*)p)[i];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = up(u.t[q]);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = q < count ? up(p[q]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void out8(T* p, const T (&t)[8], int count) {
  if (count >= 8) {
    union { words4 w[sizeof(T) / 2]; T t[8]; } u;
#pragma unroll
    for (int q = 0; q < 8; ++q) u.t[q] = t[q];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((words4*)p)[i] = u.w[i];
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < count) p[q] = t[q];
  }
}

// z + bias -> act -> + residual -> y, and z for the backward pass
template <typename T>
struct LinearOut {
  using Z = typename KeptZ<T>::Z;
  const T *bias, *res;
  T* y;
  Z* z;
  int64_t ldr, n;
  int act;
  __device__ __forceinline__ void one(float v, int64_t m, int64_t c) const {
    v += bias ? up(bias[c]) : 0.f;
    if (z) z[m * n + c] = keep_z<Z>(v);
    y[m * n + c] = down<T>(act_value(v, act) + (res ? up(res[m * ldr + c]) : 0.f));
  }
  // v: sums at row m, columns c ..; b: their bias
  __device__ __forceinline__ void eight(float (&v)[8], const float (&b)[8], int64_t m, int64_t c, int) const {
    const int count = (int)(n - c < 8 ? n - c : 8);
    if (count <= 0) return;
    float r[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (res) get8(res + m * ldr + c, r, count);
    T t[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += b[q];
    if (z) {
      Z k[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) k[q] = keep_z<Z>(v[q]);
      out8(z + m * n + c, k, count);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) t[q] = down<T>(act_value(v[q], act) + r[q]);
    out8(y + m * n + c, t, count);
  }
};

// out[order ? order[m] : m] = alpha (sum + add)
template <typename T>
struct StoreOut {
  const T* bias;  // none
  T* out;
  const float *add, *alpha;  // add: [m][n] fp32 of the pieces before
  const int32_t* order;
  int64_t n;
  __device__ __forceinline__ void eight(float (&v)[8], const float (&)[8], int64_t m, int64_t c, int) const {
    const int count = (int)(n - c < 8 ? n - c : 8);
    if (count <= 0) return;
    if (add) {
      float a[8];
      get8(add + m * n + c, a, count);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += a[q];
    }
    const float s = alpha ? *alpha : 1.f;
    T t[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) t[q] = down<T>(v[q] * s);
    out8(out + (order ? (int64_t)order[m] : m) * n + c, t, count);
  }
};

// part[split][m][n8] = sum over this block's share of k (n8: n up to 8)
struct PartOut {
  const float* bias;  // none
  float* part;
  int64_t m_all, n8;
  __device__ __forceinline__ void eight(float (&v)[8], const float (&)[8], int64_t m, int64_t c, int split) const {
    if (c < n8) out8(part + ((int64_t)split * m_all + m) * n8 + c, v, 8);
  }
};

// bias of the tile's columns in LDS as fp32
template <typename T>
__device__ __forceinline__ void stage_bias(const T* bias, int64_t n0, int64_t n, int cols, char* lds) {
  for (int c = threadIdx.x; c < cols; c += blockDim.x) ((float*)lds)[c] = bias && n0 + c < n ? up(bias[n0 + c]) : 0.f;
}

// Sums handed on in rows: 64 rows of a wave at a time go through its LDS, so that 4 TN neighbouring lanes hold 8 columns each of one row and
// loads and stores are 16 bytes wide; one loop then does whatever there is to do, where the registers' own order would need the code
// once per register (cold instructions cost a one-tile launch more than its products).
template <class Out, int BN>
struct EpiRows {
  static constexpr bool kThroughLds = true;
  Out o;
  int64_t n;
  __device__ __forceinline__ void prepare(int64_t n0, char* lds) const { stage_bias(o.bias, n0, n, BN, lds); }
  template <int TM, int TN>
  __device__ __forceinline__ void rows(f32x16 (&acc)[TM][TN], int64_t m_first, int64_t m_end, int64_t nw, int at, int split, int lane, const char* bias, char* lds) const {
    constexpr int kRow = 32 * TN + 4, kLanes = 4 * TN, kStep = 64 / kLanes, kAtOnce = TM > 1 ? 2 : 1;
    static_assert(TM % kAtOnce == 0, "whole turns");
    float* mine = (float*)lds;
    const int c = (lane % kLanes) * 8;
    float b[8];
    *(float4*)b = *(const float4*)(bias + (at + c) * 4);
    *(float4*)(b + 4) = *(const float4*)(bias + (at + c) * 4 + 16);
#pragma unroll 1
    for (int turn = 0; turn < TM / kAtOnce; ++turn) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < TM; ++j)
        if (j / kAtOnce == turn)
#pragma unroll
          for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *(float4*)(mine + (j % kAtOnce * 32 + (lane & 31)) * kRow + 32 * i + 8 * q + 4 * (lane >> 5)) =
                  float4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
      __builtin_amdgcn_wave_barrier();
      const int64_t m0 = m_first + turn * 32 * kAtOnce;
#pragma unroll 1
      for (int r = lane / kLanes; r < 32 * kAtOnce; r += kStep) {
        float v[8];
        *(float4*)v = *(const float4*)(mine + r * kRow + c);
        *(float4*)(v + 4) = *(const float4*)(mine + r * kRow + c + 4);
        if (m0 + r < m_end) o.eight(v, b, m0 + r, nw + c, split);
      }
    }
  }
};

// the splits' sums joined in their order and handed on: 8 columns a thread, G threads of a block share them by split
template <typename T, class Out, int G>
__global__ void __launch_bounds__(256) k_join(const float* part, int splits, int64_t m, int64_t n8, const int32_t* live, Out o) {
  __shared__ float sums[G][256 / G][9];
  const int64_t rows = live && *live < m ? *live : m, per = n8 / 8;
  const int t = threadIdx.x % (256 / G), g = threadIdx.x / (256 / G), share = (splits + G - 1) / G;
  const int from = g * share, to = from + share < splits ? from + share : splits;
  for (int64_t i0 = (int64_t)blockIdx.x * (256 / G); i0 < rows * per; i0 += (int64_t)gridDim.x * (256 / G)) {
    const int64_t i = i0 + t, r = i / per, c = (i - r * per) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (i < rows * per)
#pragma unroll 4
      for (int s = from; s < to; ++s) {
        const float4* p = (const float4*)(part + ((int64_t)s * m + r) * n8 + c);
        const float4 a = p[0], b = p[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
    if constexpr (G > 1) {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 8; ++q) sums[g][t][q] = v[q];
      __syncthreads();
      if (g) continue;
      for (int s = 1; s < G; ++s)
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] += sums[s][t][q];
    }
    if (i >= rows * per) continue;
    float b[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) b[q] = o.bias && c + q < o.n ? up(o.bias[c + q]) : 0.f;
    o.eight(v, b, r, c, 0);
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
  static constexpr bool kThroughLds = false;
  __device__ __forceinline__ void prepare(int64_t n0, char* lds) const { stage_bias(bias, n0, n, BN, lds); }
  template <int TM, int TN>
  __device__ __forceinline__ void rows(f32x16 (&acc)[TM][TN], int64_t m_first, int64_t m_end, int64_t nw, int at, int, int lane, const char* lds, char*) const {
#pragma unroll
    for (int j = 0; j < TM; ++j) row<TN>(acc[j], m_first + 32 * j, m_end, nw, at, lane, lds);
  }
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t m_first, int64_t m_end, int64_t nw, int at, int lane, const char* lds) const {
    if (nw >= n) return;
    const int half = lane >> 5;
    const int64_t m = m_first + (lane & 31);
    const bool on = m < m_end;
    if (bias) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 b = *(const float4*)(lds + (at + 32 * i + 8 * j + 4 * half) * 4);
          acc[i][4 * j] += b.x; acc[i][4 * j + 1] += b.y; acc[i][4 * j + 2] += b.z; acc[i][4 * j + 3] += b.w;
        }
    }
    if (nw + 32 * TN > n) {  // columns that are not there
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (nw + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3) >= n) acc[i][r] = neg_inf();
    }
    if constexpr (!LABEL) {
      const int64_t tt = on ? target[order[m]] - nw : -1;
      const int t = tt >= 0 && tt < 32 * TN ? (int)tt : -1;
      if (__any(t >= 0)) {  // few waves hold a target of theirs
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (t == 32 * i + 8 * (r >> 2) + 4 * half + (r & 3)) zt[m] = acc[i][r];
      }
    }
    float top = neg_inf();
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float safe = top == neg_inf() ? 0.f : top;
    // sum of all exp(z - top), the largest one's 1 among them; where the others are less than half of it that sum has lost more of their last
    // bits than a sum loses anyway, and they are added up again without it (down to 2^-6 only, which lost 6 bits: 8192 x 2048 -> 65536 bf16
    // 1.67 ms either way, 1048576 x 64 -> 72 fp16 with random logits 0.21 and 0.22)
    float rest = 0.f;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) rest += __builtin_amdgcn_exp2f((acc[i][r] - safe) * 1.4426950408889634f);
    rest += __shfl_xor(rest, 32, 64);
    rest -= 1.f;
    if (__any(!(rest >= 0.5f))) {
      float again = 0.f;
      int same = 0;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool is = acc[i][r] == top;
          again += is ? 0.f : __builtin_amdgcn_exp2f((acc[i][r] - safe) * 1.4426950408889634f);
          same += is;
        }
      again += __shfl_xor(again, 32, 64);
      same += __shfl_xor(same, 32, 64);
      if (!(rest >= 0.5f)) rest = again + (float)(same - 1);
    }
    if (top == neg_inf()) rest = rest == rest ? 0.f : rest;  // nothing finite here: a join counts nothing
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
      if (__any(odd)) {
        int first = 0x7fffffff;
#pragma unroll
        for (int i = TN - 1; i >= 0; --i)
#pragma unroll
          for (int r = 15; r >= 0; --r)
            if (acc[i][r] != acc[i][r]) first = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
        const int other = __shfl_xor(first, 32, 64);
        first = other < first ? other : first;
        nan = odd && first != 0x7fffffff;
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

// v[e] of the 32 lanes of each half of a wave added up: lane l keeps the sum of element l % 32 of 32, or l % 32 / 2 of 16.  Each step halves what
// a lane still holds: it gives away one half and adds up the other.
template <int N, int COUNT = N, int D = 16>
__device__ __forceinline__ float half_wave_sums(float (&v)[N], int lane) {
  static_assert(N == 16 || N == 32, "elements a lane");
  if constexpr (D == 0) {
    return v[0];
  } else if constexpr (COUNT > 1) {
    const bool upper = lane & D;
#pragma unroll
    for (int e = 0; e < COUNT / 2; ++e) {
      const float keep = upper ? v[e + COUNT / 2] : v[e], give = upper ? v[e] : v[e + COUNT / 2];
      v[e] = keep + __shfl_xor(give, D, 64);
    }
    return half_wave_sums<N, COUNT / 2, D / 2>(v, lane);
  } else {
    v[0] += __shfl_xor(v[0], D, 64);
    return half_wave_sums<N, 1, D / 2>(v, lane);
  }
}

// dz of a piece of the classes, in NP planes: (p - onehot) x the row's factor; and for db its column sums over the wave's rows, before it is
// rounded (of dz in bf16 they are off by up to 2^-9 of sum |dz|, much more than a rounding of db where its terms cancel;
// 8192 x 2048 -> 65536 bf16: 1.10 ms a piece with them, 1.09 without, where a pass over the piece's dz takes 0.12)
template <typename T, int BN, int NP>
struct EpiDz {
  const T* bias;  // of the piece
  const int64_t* target;
  const int32_t* order;
  const float4* stat;  // [row in order]
  const float* scale;  // [0]: what every row is multiplied by
  const float* g;      // per-row factor, by original row, or NULL
  uint16_t* dz;
  float* sums;  // [run of 32 TM rows][n], or NULL
  int64_t v0, n, ld;  // columns v0 .. v0 + n; ld: n padded (zeros there)
  static constexpr bool kThroughLds = false;
  __device__ __forceinline__ void prepare(int64_t n0, char* lds) const { stage_bias(bias, n0, n, BN, lds); }
  template <int TM, int TN>
  __device__ __forceinline__ void rows(f32x16 (&acc)[TM][TN], int64_t m_first, int64_t m_end, int64_t nw, int at, int, int lane, const char* lds, char*) const {
    if (m_first >= m_end) return;
    float v[16 * TN];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      row<TN>(acc[j], m_first + 32 * j, m_end, nw, at, lane, lds);
#pragma unroll
      for (int e = 0; e < 16 * TN; ++e) v[e] = (j ? v[e] : 0.f) + acc[j][e / 16][e % 16];
    }
    if (!sums || nw >= n) return;
    const float sum = half_wave_sums(v, lane);
    const int e = TN == 2 ? lane & 31 : (lane & 31) >> 1, c = 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * (lane >> 5) + (e & 3);
    if (nw + c < n && (TN == 2 || (lane & 1) == 0)) sums[m_first / (32 * TM) * n + nw + c] = sum;
  }
  // acc becomes dz, zeros in rows that are not there
  template <int TN>
  __device__ __forceinline__ void row(f32x16 (&acc)[TN], int64_t m_first, int64_t m_end, int64_t nw, int at, int lane, const char* lds) const {
    const int half = lane >> 5;
    const bool on = m_first + (lane & 31) < m_end;
    const int64_t m = on ? m_first + (lane & 31) : m_end - 1;  // rows that are not there: zeros
    const int64_t from = order[m];
    const float4 s = stat[m];
    const int64_t tt = target[from] - v0 - nw;
    const int t = tt >= 0 && tt < 32 * TN && tt < n - nw ? (int)tt : -1;  // (a class that is not there: the row is NaN by stat)
    float f = scale[0];
    if (g) f *= g[from];
    const float inv = s.w != s.w ? s.w : s.y * f, hit = s.z * f;
    const bool tail = nw + 32 * TN > n;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * i + 8 * j + 4 * half;
        if (tail && nw + c >= ld) continue;
        if (bias) {
          const float4 b = *(const float4*)(lds + (at + c) * 4);
          acc[i][4 * j] += b.x; acc[i][4 * j + 1] += b.y; acc[i][4 * j + 2] += b.z; acc[i][4 * j + 3] += b.w;
        }
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = __builtin_amdgcn_exp2f((acc[i][4 * j + q] - s.x) * 1.4426950408889634f) * inv;
          v[q] = t == c + q ? hit : v[q];
          if (!on) v[q] = 0.f;
        }
        if (tail) {
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = nw + c + q < n ? v[q] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][4 * j + q] = v[q];
        if (on) put(dz + m * ld * NP + column<NP>(nw) + (NP == 3 ? 96 * i + 8 * j + 4 * half : c), v);
      }
  }
  __device__ __forceinline__ void put(uint16_t* to, const float (&v)[4]) const {
    if constexpr (NP == 1) {
      union { uint16_t w[4]; T t[4]; } u;
#pragma unroll
      for (int q = 0; q < 4; ++q) u.t[q] = down<T>(v[q]);
      *(ushort4*)to = ushort4{u.w[0], u.w[1], u.w[2], u.w[3]};
    } else {
      uint16_t h[4][3];
#pragma unroll
      for (int q = 0; q < 4; ++q) planes(v[q], h[q]);
#pragma unroll
      for (int s3 = 0; s3 < 3; ++s3) *(ushort4*)(to + s3 * 32) = ushort4{h[0][s3], h[1][s3], h[2][s3], h[3][s3]};
    }
  }
};

}  // namespace clid_dense
