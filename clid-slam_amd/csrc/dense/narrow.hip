// The dense operators at a point decoder's own widths, n <= 64 and k <= 64: memory bound, so x is read once and everything else happens in
// registers.
//
// A wave takes 32 rows at a time; the weight lies in LDS.  z = x w^T on the matrix instruction of x's type, with the rows of w as its row operand:
// a lane then holds one row m of x and of z, element (i, r) being column 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4.  (32 x 32 x 2 for fp32;
// 32 x 32 x 16 for 16 bits: 1048576 x 64 -> 64 bf16 gelu 87 us, 3.1 TB/s, label 50, and 140 and 106 by the fp32 one, whose products take 16 times
// as long.  fp32 as bf16 planes, as the tiles have it: 1048576 x 64 -> 21 label 87 us, 70 by the fp32 instruction, as splitting x costs more than the
// products.)  A row's softmax is 16 or 32 registers and one exchange between two lanes, with no partial results in memory.  The same
// registers are the column operand of dx = dz w as they are (fp32 instruction; the contraction over n takes its columns in that order, and so
// does the row operand, read from w in LDS).  dw = dz^T x contracts over m: dz goes through LDS once, x is there already; the sums over a
// wave's rows stay in accumulators, a block's waves add theirs in LDS, k_narrow_join adds the blocks' in their order.  Nothing is
// rounded before the results, whatever the type.  The cross entropy's backward pass makes z again rather than keeping anything of it.
//
// x comes by 16-byte copies straight to LDS, the next 32 rows' while these are worked on; chunks are permuted within their row so that the
// lanes' reads fall on different banks.  (By 16-byte loads to registers, each of 32 rows' 32 bytes: 1048576 x 64 -> 21 fp32 label 140 us, 77 us
// this way.)  Rows that are not whole aligned chunks (11 features) come through registers all the same.
#include "stage.hpp"

namespace clid_dense {

typedef __attribute__((ext_vector_type(16))) float f32x16;

enum class Do { Linear, LinearBwd, Ce, CeBwd, Label };

struct Narrow {
  const void *x, *w, *bias;
  int64_t ldx, ldw, rows;
  int k, n, x_wide, work;  // work: waves of a block that take rows; the others help with w and with the sums
  // Linear, LinearBwd
  const void *res, *dy, *z_in;
  void *y, *z_out;
  int64_t ldr, lddy;
  int act, z_is_y;
  // LinearBwd, CeBwd
  void* dx;
  float* part;  // [blocks][n k + n]: sums for dw and db
  int want_w;
  // Ce, CeBwd
  const int64_t* target;
  int64_t ignore;
  int reduction;
  float *loss_none, *total;
  const float* g;
  double* sums;  // [blocks][2]: losses, how many
  // Label
  int64_t* label;
  float* log_prob;
};

__device__ __forceinline__ f32x16 mfma_f32(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// 32 rows of 32 T fp32 values in a wave's LDS, 16-byte chunks permuted within the row.  The products leave them lane by row (a lane holds row
// lane % 32, chunks 8 i + 2 j + lane / 32); memory wants them 8 neighbouring values a lane.
template <int T>
struct Rows32 {
  static __device__ __forceinline__ float* chunk(float* tile, int row, int c) { return tile + row * 32 * T + (c ^ (row & (8 * T - 1))) * 4; }
  static __device__ __forceinline__ void put(float* tile, const f32x16 (&v)[T], int lane) {
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(float4*)chunk(tile, lane & 31, 8 * i + 2 * j + (lane >> 5)) = float4{v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3]};
  }
  static __device__ __forceinline__ void get(float* tile, f32x16 (&v)[T], int lane) {
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 f = *(const float4*)chunk(tile, lane & 31, 8 * i + 2 * j + (lane >> 5));
        v[i][4 * j] = f.x; v[i][4 * j + 1] = f.y; v[i][4 * j + 2] = f.z; v[i][4 * j + 3] = f.w;
      }
  }
  // f(row, first column, 8 values) over the tile: one copy of its code, 4 T neighbouring lanes a row
  template <class F>
  static __device__ __forceinline__ void each8(float* tile, int lane, const F& f) {
    const int c = lane % (4 * T);
#pragma unroll 1
    for (int row = lane / (4 * T); row < 32; row += 16 / T) {
      float v[8];
      float *lo = chunk(tile, row, 2 * c), *hi = chunk(tile, row, 2 * c + 1);
      *(float4*)v = *(const float4*)lo;
      *(float4*)(v + 4) = *(const float4*)hi;
      f(row, 8 * c, v, lo, hi);
    }
  }
};

// f with the activation as a constant of its type: one branch where many values have the same
template <class F>
__device__ __forceinline__ void by_act(int act, const F& f) {
  switch (act) {
    case CLID_ACT_RELU: return f(std::integral_constant<int, CLID_ACT_RELU>{});
    case CLID_ACT_LEAKY_RELU: return f(std::integral_constant<int, CLID_ACT_LEAKY_RELU>{});
    case CLID_ACT_GELU: return f(std::integral_constant<int, CLID_ACT_GELU>{});
    case CLID_ACT_SILU: return f(std::integral_constant<int, CLID_ACT_SILU>{});
    default: return;
  }
}

// TN: 32 columns of z each; KQ: runs of 8 along k
template <typename T, int TN, int KQ, Do DO>
struct NarrowShape {
  static constexpr int max_of(int a, int b) { return a > b ? a : b; }
  static constexpr bool kBwd = DO == Do::LinearBwd || DO == Do::CeBwd;
  static constexpr int kChunkElems = 16 / sizeof(T);
  static constexpr int kChunks = 8 * KQ / kChunkElems;             // of an x row in LDS: 2, 4, 8 or 16
  static constexpr int kTK = (8 * KQ + 31) / 32;
  static constexpr int kXLoads = 32 * kChunks * 16 / 1024;
  // 32 rows; the same place then holds 32 rows of y on their way out
  static constexpr int kXBuf = max_of(32 * kChunks * 16, DO == Do::Linear ? 32 * TN * 128 : 0);
  // Backward passes have one place for x (the next rows' copy starts when dw has read these, and runs under dx), so that 8 waves fit a CU and one
  // multiplies while another waits.  1048576 x 64 -> 64 fp32, forward and backward: cross entropy 523 us with 4 waves and two places, 415 this
  // way, a layer with gelu 639 and 440.
  static constexpr int kXBufs = kBwd ? 1 : 2;
  static constexpr int kMostWaves = 8;
  static constexpr int kWRow = 8 * KQ + kChunkElems;               // elements: rows that are read together start on different banks
  static constexpr int kWBytes = 32 * TN * kWRow * (int)sizeof(T);
  static constexpr int kZBytes = kBwd ? 32 * 32 * max_of(TN, kTK) * 4 : 0;  // dz, then dx on its way out
  static constexpr int kWave = kXBufs * kXBuf + kZBytes;
  static constexpr int kHead = kWBytes + 32 * TN * 4;
  static constexpr int kSumRow = 32 * kTK + 1, kSums = 32 * TN * kSumRow + 32 * TN;  // a wave's sums for dw and db, floats
  static constexpr int lds(int work) { return max_of(kHead + work * kWave, kBwd ? work * kSums * 4 : kMostWaves * 16); }
  // 16 chunks span the banks once: the rows between them are told apart by the chunk's place
  static __device__ __forceinline__ int place(int row, int c) { return c ^ ((row / (16 / kChunks)) & (kChunks - 1)); }
};

template <typename T, int TN, int KQ, Do DO>
__global__ void __launch_bounds__(512) k_narrow(Narrow a) {
  using S = NarrowShape<T, TN, KQ, DO>;
  constexpr int TK = S::kTK;
  extern __shared__ __align__(16) char lds[];
  T* w = (T*)lds;
  float* bias = (float*)(lds + S::kWBytes);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int waves = blockDim.x >> 6;
  char* xbuf = lds + S::kHead + wave * S::kWave;
  float* zbuf = (float*)(xbuf + S::kXBufs * S::kXBuf);
  const T* x = (const T*)a.x;

  // copies' offsets, the same for every 32 rows
  uint32_t at[S::kXLoads];
#pragma unroll
  for (int i = 0; i < S::kXLoads; ++i) {
    const int c = i * 64 + lane, row = c / S::kChunks, chunk = S::place(row, c % S::kChunks);
    at[i] = chunk * S::kChunkElems < a.k ? uint32_t(row) * uint32_t(a.ldx * sizeof(T)) + chunk * 16 : kOutside;
  }
  auto fetch = [&](int64_t m0, char* buf) {
    const int64_t rows = a.rows - m0 < 32 ? a.rows - m0 : 32;
    if (a.x_wide) {
      const uint32_t bound = (uint32_t)(((rows - 1) * a.ldx + a.k) * (int64_t)sizeof(T));
#pragma unroll
      for (int i = 0; i < S::kXLoads; ++i) copy16(x + m0 * a.ldx, bound, at[i], buf + i * 1024);
    } else {
      constexpr int kEach = 8 * KQ / 2;  // two lanes a row
      const T* from = x + (m0 + col) * a.ldx;
      T v[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) v[e] = col < rows && half * kEach + e < a.k ? from[half * kEach + e] : down<T>(0.f);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int k = half * kEach + e;
        ((T*)(buf + (col * S::kChunks + S::place(col, k / S::kChunkElems)) * 16))[k % S::kChunkElems] = v[e];
      }
    }
  };

  const int64_t strips = (a.rows + 31) / 32, step = (int64_t)gridDim.x * a.work;
  int64_t strip = wave < a.work ? (int64_t)blockIdx.x * a.work + wave : strips;
  if (a.x_wide && strip < strips) fetch(strip * 32, xbuf);
#pragma unroll 4
  for (int e = threadIdx.x; e < 32 * TN * KQ; e += blockDim.x) {  // 8 values each
    const int n = e / KQ, k = e % KQ * 8;
    float v[8];
    get8((const T*)a.w + n * a.ldw + k, v, n < a.n ? a.k - k : 0);
    struct alignas(16) Run { T t[8]; } run;
#pragma unroll
    for (int q = 0; q < 8; ++q) run.t[q] = down<T>(v[q]);
    *(Run*)(w + n * S::kWRow + k) = run;
  }
  for (int n = threadIdx.x; n < 32 * TN; n += blockDim.x) bias[n] = a.bias && n < a.n ? up(((const T*)a.bias)[n]) : 0.f;
  __syncthreads();

  f32x16 sum_w[S::kBwd ? TN : 1][S::kBwd ? TK : 1];
  float sum_b[TN];  // column 32 i + lane % 32, every other row
  if constexpr (S::kBwd) {
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      sum_b[i] = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int t = 0; t < TK; ++t) sum_w[i][t][r] = 0.f;
    }
  }
  double loss_sum = 0.0;
  int counted = 0;

  for (int turn = 0; strip < strips; strip += step, turn ^= 1) {
    // Backward passes: LDS addresses are made anew each turn.  Kept from one turn to the next, as the compiler would, they take 100 registers and
    // other values are spilled for them.
    int here = threadIdx.x & 63;
    if constexpr (S::kBwd) asm volatile("" : "+v"(here));
    const int lane = here, col = lane & 31, half = lane >> 5;
    char* xs = S::kXBufs == 2 ? xbuf + turn * S::kXBuf : xbuf;
    const int64_t m0 = strip * 32, m = m0 + col;
    const bool on = m < a.rows;
    if (!a.x_wide) fetch(m0, xs);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // these rows' copies; no read of them moves above it
    if (S::kXBufs == 2 && a.x_wide && strip + step < strips) fetch((strip + step) * 32, xbuf + (turn ^ 1) * S::kXBuf);

    f32x16 z[TN];
    if constexpr (DO != Do::LinearBwd) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 b4 = *(const float4*)(bias + 32 * i + 8 * j + 4 * half);
          z[i][4 * j] = b4.x; z[i][4 * j + 1] = b4.y; z[i][4 * j + 2] = b4.z; z[i][4 * j + 3] = b4.w;
        }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int q = 0; q < KQ; q += 2) {
          const s16x8 xv = *(const s16x8*)(xs + (col * S::kChunks + S::place(col, q + half)) * 16);
#pragma unroll
          for (int i = 0; i < TN; ++i) z[i] = mfma<Kind<T>::F16>(*(const s16x8*)(w + (32 * i + col) * S::kWRow + 8 * (q + half)), xv, z[i]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < KQ; ++q) {  // 8 q + 4 half ..
          const float4 x4 = *(const float4*)(xs + (col * S::kChunks + S::place(col, 2 * q + half)) * 16);
#pragma unroll
          for (int i = 0; i < TN; ++i) {
            const float4 w4 = *(const float4*)(w + (32 * i + col) * S::kWRow + 8 * q + 4 * half);
            z[i] = mfma_f32(w4.x, x4.x, z[i]);
            z[i] = mfma_f32(w4.y, x4.y, z[i]);
            z[i] = mfma_f32(w4.z, x4.z, z[i]);
            z[i] = mfma_f32(w4.w, x4.w, z[i]);
          }
        }
      }
    }

    if constexpr (DO == Do::Linear) {
      const LinearOut<T> o = {nullptr, (const T*)a.res, (T*)a.y, (typename KeptZ<T>::Z*)a.z_out, a.ldr, a.n, a.act};
      float* tile = (float*)xs;  // x is done with
      Rows32<TN>::put(tile, z, lane);
      __builtin_amdgcn_wave_barrier();
      Rows32<TN>::each8(tile, lane, [&](int row, int c, float (&v)[8], float*, float*) {
        const float none[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // the bias is in z
        if (m0 + row < a.rows) o.eight(v, none, m0 + row, c, 0);
      });
      __builtin_amdgcn_wave_barrier();
    }

    // a row's statistics: the largest z, its column, sum over the others of exp(z - largest), the target's z
    float top = neg_inf(), rest = 0.f, zt = 0.f;
    int best = 0x7fffffff;
    bool counts = false;
    int64_t target = -1;
    if constexpr (DO == Do::Ce || DO == Do::CeBwd) {
      if (on) target = a.target[m];
      counts = on && target != a.ignore;
    }
    if constexpr (DO == Do::Ce || DO == Do::CeBwd || DO == Do::Label) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
          if (n >= a.n) z[i][r] = neg_inf();
          if (n == target) zt = z[i][r];
          top = fmaxf(top, z[i][r]);
        }
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float safe = top == neg_inf() ? 0.f : top;
      int same = 0;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool is = z[i][r] == top;
          rest += is ? 0.f : __builtin_amdgcn_exp2f((z[i][r] - safe) * 1.4426950408889634f);
          same += is;
        }
      rest += __shfl_xor(rest, 32, 64);
      same += __shfl_xor(same, 32, 64);
      zt += __shfl_xor(zt, 32, 64);  // the other half's is 0
      rest = top == neg_inf() ? (rest == rest ? 0.f : rest) : rest + (float)(same - 1);
      if (top == __builtin_inff()) rest = __builtin_nanf("");
    }
    float loss = 0.f;
    if constexpr (DO == Do::Ce || DO == Do::CeBwd) {
      loss = target >= 0 && target < a.n ? (top - zt) + log1pf(rest) : __builtin_nanf("");
      if (!counts) loss = 0.f;
    }
    if constexpr (DO == Do::Ce) {
      if (half == 0 && on) {
        if (a.loss_none) a.loss_none[m] = loss;
        loss_sum += loss;
        counted += counts;
      }
    }
    if constexpr (DO == Do::Label) {
      bool nan = false;
#pragma unroll
      for (int i = TN - 1; i >= 0; --i)
#pragma unroll
        for (int r = 15; r >= 0; --r)
          if (z[i][r] == top) best = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
      if (rest != rest) {
        int first = 0x7fffffff;
#pragma unroll
        for (int i = TN - 1; i >= 0; --i)
#pragma unroll
          for (int r = 15; r >= 0; --r)
            if (z[i][r] != z[i][r]) first = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
        const int other = __shfl_xor(first, 32, 64);
        first = other < first ? other : first;
        nan = first != 0x7fffffff;
        if (nan) best = first;
      }
      const int other = __shfl_xor(best, 32, 64);
      best = other < best ? other : best;
      if (half == 0 && on) {
        a.label[m] = best;
        a.log_prob[m] = nan || top == neg_inf() ? __builtin_nanf("") : -log1pf(rest);
      }
    }

    if constexpr (S::kBwd) {
      // z becomes dz
      if constexpr (DO == Do::LinearBwd) {
        // all loads first
        constexpr int kEach = 2 * TN;
        const int c = lane % (4 * TN) * 8;
        float v[kEach][8], y[kEach][8];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int64_t at = m0 + lane / (4 * TN) + e * (16 / TN);
          const int count = at < a.rows ? a.n - c : 0;
          get8((const T*)a.dy + at * a.lddy + c, v[e], count);
          if (!a.z_in) continue;
          if (a.z_is_y) get8((const T*)a.z_in + at * a.n + c, y[e], count);
          else get8((const typename KeptZ<T>::Z*)a.z_in + at * a.n + c, y[e], count);
        }
        if (a.z_in) by_act(a.act, [&](auto act) {
#pragma unroll
          for (int e = 0; e < kEach; ++e)
#pragma unroll
            for (int q = 0; q < 8; ++q)
              v[e][q] = m0 + lane / (4 * TN) + e * (16 / TN) < a.rows && c + q < a.n ? act_grad(v[e][q], y[e][q], act) : 0.f;
        });
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int row = lane / (4 * TN) + e * (16 / TN);
          *(float4*)Rows32<TN>::chunk(zbuf, row, c / 4) = *(const float4*)v[e];
          *(float4*)Rows32<TN>::chunk(zbuf, row, c / 4 + 1) = *(const float4*)(v[e] + 4);
        }
        __builtin_amdgcn_wave_barrier();
        Rows32<TN>::get(zbuf, z, lane);
      } else {
        float f = 0.f;
        if (counts) f = a.reduction == CLID_REDUCE_NONE ? a.g[m] : a.reduction == CLID_REDUCE_MEAN ? a.g[0] / fmaxf(a.total[1], 1.f) : a.g[0];
        const float inv = loss != loss ? loss : f / (1.f + rest), hit = expm1f(-loss) * f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int n = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
            const float p = __builtin_amdgcn_exp2f((z[i][r] - top) * 1.4426950408889634f) * inv;
            z[i][r] = counts && n < a.n ? (n == target ? hit : p) : 0.f;
          }
      }
      if constexpr (DO == Do::CeBwd) Rows32<TN>::put(zbuf, z, lane);
      __builtin_amdgcn_wave_barrier();
      // rows that do not count are zeros whatever they hold
      const uint32_t live = DO == Do::CeBwd ? (uint32_t)__ballot(counts) : 0xffffffffu;
#pragma unroll
      for (int s = 0; s < 16; ++s) {
        const int mm = 2 * s + half;
        float zv[TN];
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          zv[i] = Rows32<TN>::chunk(zbuf, mm, 8 * i + (col >> 2))[col & 3];
          sum_b[i] += zv[i];
        }
        if (!a.want_w) continue;
        float xv[TK];
#pragma unroll
        for (int t = 0; t < TK; ++t) {
          const int k = 32 * t + col;
          xv[t] = 0.f;
          if ((8 * KQ >= 32 || k < 8 * KQ) && (live >> mm & 1)) xv[t] = up(((const T*)(xs + (mm * S::kChunks + S::place(mm, k / S::kChunkElems)) * 16))[k % S::kChunkElems]);
        }
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int t = 0; t < TK; ++t) sum_w[i][t] = mfma_f32(zv[i], xv[t], sum_w[i][t]);
      }
      if (a.x_wide && strip + step < strips) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // nothing reads these rows any more
        fetch((strip + step) * 32, xs);
      }
      if (a.dx) {
        f32x16 d[TK];
#pragma unroll
        for (int t = 0; t < TK; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) d[t][r] = 0.f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int n = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
            for (int t = 0; t < TK; ++t) {
              const int k = 32 * t + col;  // a row of w is 8 KQ values: where that is 16, lanes 16 .. 31 have none
              d[t] = mfma_f32(8 * KQ >= 32 || k < 8 * KQ ? up(w[n * S::kWRow + k]) : 0.f, z[i][r], d[t]);
            }
          }
        __builtin_amdgcn_wave_barrier();
        Rows32<TK>::put(zbuf, d, lane);  // dw is done with dz
        __builtin_amdgcn_wave_barrier();
        Rows32<TK>::each8(zbuf, lane, [&](int row, int c, float (&v)[8], float*, float*) {
          if (m0 + row >= a.rows) return;
          const bool zero = DO == Do::CeBwd && !(live >> row & 1);
          T t[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) t[q] = down<T>(zero ? 0.f : v[q]);
          out8((T*)a.dx + (m0 + row) * a.k + c, t, a.k - c);
        });
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  if constexpr (DO == Do::Ce) {
    for (int d = 16; d; d >>= 1) {
      loss_sum += __shfl_xor(loss_sum, d, 64);
      counted += __shfl_xor(counted, d, 64);
    }
    __syncthreads();
    double* s = (double*)lds;
    if (lane == 0) {
      s[2 * wave] = loss_sum;
      s[2 * wave + 1] = counted;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      double t = 0.0;
      for (int i = 0; i < waves; ++i) t += s[2 * i + threadIdx.x];
      a.sums[blockIdx.x * 2 + threadIdx.x] = t;
    }
  }
  if constexpr (S::kBwd) {
    // the waves' sums: [wave][n][k] and [wave][n], then one partial result a block
    __syncthreads();
    constexpr int kRow = S::kSumRow, kMine = S::kSums;
    float* mine = (float*)lds + wave * kMine;
    if (wave < a.work)
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const float b = sum_b[i] + __shfl_xor(sum_b[i], 32, 64);
        if (half == 0) mine[32 * TN * kRow + 32 * i + col] = b;
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int t = 0; t < TK; ++t) mine[(32 * i + 8 * (r >> 2) + 4 * half + (r & 3)) * kRow + 32 * t + col] = sum_w[i][t][r];
      }
    __syncthreads();
    const float* all = (const float*)lds;
    float* out = a.part + (int64_t)blockIdx.x * (a.n * a.k + a.n);
    const auto total = [&](int from) {
      float t = 0.f;
      for (int i = 0; i < a.work; ++i) t += all[i * kMine + from];
      return t;
    };
    if (a.want_w)
#pragma unroll 4
      for (int e = threadIdx.x; e < a.n * 32 * TK; e += blockDim.x) {
        const int n = e / (32 * TK), k = e % (32 * TK);
        if (k < a.k) out[n * a.k + k] = total(n * kRow + k);
      }
    for (int n = threadIdx.x; n < a.n; n += blockDim.x) out[a.n * a.k + n] = total(32 * TN * kRow + n);
  }
}

// the blocks' sums -> dw, db: 64 of them a block, 16 threads each
template <typename T>
__global__ void __launch_bounds__(1024) k_narrow_join(const float* part, int blocks, int nk, int n, T* dw, T* db) {
  __shared__ float p[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6, all = nk + n;
  float s = 0.f;
  if (c < nk ? dw != nullptr : c < all)  // (without dw nothing was left of it)
#pragma unroll 8
    for (int b = g; b < blocks; b += 16) s += part[(int64_t)b * all + c];
  p[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g || c >= all) return;
  for (int i = 1; i < 16; ++i) s += p[i][threadIdx.x];
  if (c < nk) {
    if (dw) dw[c] = down<T>(s);
  } else if (db) {
    db[c - nk] = down<T>(s);
  }
}
__global__ void __launch_bounds__(256) k_narrow_total(const double* sums, int blocks, int reduction, float* total, float* loss_out) {
  __shared__ double p[4][2];
  double s = 0.0, c = 0.0;
  for (int b = threadIdx.x; b < blocks; b += 256) {
    s += sums[2 * b];
    c += sums[2 * b + 1];
  }
  for (int d = 32; d; d >>= 1) {
    s += __shfl_xor(s, d, 64);
    c += __shfl_xor(c, d, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    p[threadIdx.x >> 6][0] = s;
    p[threadIdx.x >> 6][1] = c;
  }
  __syncthreads();
  if (threadIdx.x) return;
  s = p[0][0] + p[1][0] + p[2][0] + p[3][0];
  c = p[0][1] + p[1][1] + p[2][1] + p[3][1];
  total[0] = (float)s;
  total[1] = (float)c;
  if (reduction == CLID_REDUCE_MEAN) loss_out[0] = c > 0.0 ? (float)(s / c) : 0.f;
  if (reduction == CLID_REDUCE_SUM) loss_out[0] = (float)s;
}

// 32 rows a wave and turn.  Where there is at most one block a CU it has all 8 waves, however few take rows: the others help to bring w and to add
// up (1000 x 64 -> 64 fp32, layer and gradients: 24 us, 44 without that and with divisions in the sums' last loop).  As many blocks as CUs (two or
// more a CU where few waves fit one): a block's copy of w serves all its turns,
// and no second round of blocks waits behind the first.  Of the waves a block may have, as many as leave the busiest CU the fewest turns:
// 98304 rows of 64 -> 64 fp32 take two turns of 6 waves (8 waves: half the CUs two turns, the others one).
struct NarrowGrid {
  int work, waves, blocks;  // waves of a block that take rows, all of them
};
template <class S>
NarrowGrid narrow_grid(int64_t rows) {
  const int64_t strips = (rows + 31) / 32;
  int waves = 1;
  int64_t least = INT64_MAX;
  for (int w = 1; w <= S::kMostWaves; ++w) {
    const int64_t turns = (strips + (int64_t)kCus * w - 1) / ((int64_t)kCus * w);
    if (turns * w <= least) {
      least = turns * w;
      waves = w;
    }
    if (turns == 1) break;
  }
  const int64_t b = (strips + waves - 1) / waves;
  int fit = 160 * 1024 / S::lds(waves);
  if (fit > 8 / waves) fit = 8 / waves;  // 8 waves a CU
  if (fit < 1) fit = 1;
  const int64_t most = (int64_t)kCus * fit;
  const int blocks = (int)(b < most ? b : most);
  return {waves, blocks <= kCus ? S::kMostWaves : waves, blocks};
}

template <typename T, int TN, int KQ, Do DO>
int narrow_launch(Narrow a, hipStream_t s) {
  using S = NarrowShape<T, TN, KQ, DO>;
  static_assert(S::lds(S::kMostWaves) <= 160 * 1024, "a block fits a CU");
  const NarrowGrid g = narrow_grid<S>(a.rows);
  auto k = k_narrow<T, TN, KQ, DO>;
  a.work = g.work;
  const int lds = S::lds(g.work), rc = allow_lds((const void*)k, S::lds(S::kMostWaves));
  if (rc != CLID_OK) return rc;
  hipLaunchKernelGGL(k, dim3(g.blocks), dim3(64 * g.waves), lds, s, a);
  return g.blocks;
}
template <typename T, Do DO>
int narrow_by_shape(const Narrow& a, hipStream_t s) {  // how many blocks, or an error
  if (a.n <= 32) {
    if (a.k <= 16) return narrow_launch<T, 1, 2, DO>(a, s);
    if (a.k <= 32) return narrow_launch<T, 1, 4, DO>(a, s);
    return narrow_launch<T, 1, 8, DO>(a, s);
  }
  if (a.k <= 16) return narrow_launch<T, 2, 2, DO>(a, s);
  if (a.k <= 32) return narrow_launch<T, 2, 4, DO>(a, s);
  return narrow_launch<T, 2, 8, DO>(a, s);
}

template <typename T>
static Narrow narrow_args(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int64_t rows, int k, int n) {
  Narrow a = {};
  a.x = x; a.w = w; a.bias = bias;
  a.ldx = ldx; a.ldw = ldw; a.rows = rows;
  a.k = k; a.n = n;
  a.x_wide = (uintptr_t)x % 16 == 0 && ldx % (16 / (int)sizeof(T)) == 0 && k % (16 / (int)sizeof(T)) == 0 && ldx < (int64_t(1) << 24);
  return a;
}
constexpr int kMostBlocks = 8 * kCus;  // of one wave each

int narrow_linear(const clid_linear_args* c, hipStream_t s) {
  int blocks = 0;
  BY_DTYPE(c->dtype, {
    Narrow a = narrow_args<T>(c->x, c->ldx, c->w, c->ldw, c->bias, c->rows, c->k, c->n);
    a.res = c->residual; a.ldr = c->ldr; a.y = c->y; a.z_out = c->z_out; a.act = c->act;
    blocks = narrow_by_shape<T, Do::Linear>(a, s);
  });
  return blocks < 0 ? blocks : CLID_OK;
}
static int64_t part_bytes_of(int64_t rows, int k, int n) {
  const int64_t strips = (rows + 31) / 32;
  return up256((strips < kMostBlocks ? strips : kMostBlocks) * ((int64_t)n * k + n) * 4);
}
template <typename T, Do DO>
static int narrow_bwd(Narrow& a, void* dw, void* db, hipStream_t s) {
  const int all = a.n * a.k + a.n, blocks = narrow_by_shape<T, DO>(a, s);
  if (blocks < 0) return blocks;
  if (dw || db) hipLaunchKernelGGL(k_narrow_join<T>, dim3((all + 63) / 64), dim3(1024), 0, s, (const float*)a.part, blocks, a.n * a.k, a.n, (T*)dw, (T*)db);
  return CLID_OK;
}
int64_t narrow_linear_bwd_bytes(const clid_linear_bwd_args* c) { return part_bytes_of(c->rows, c->k, c->n); }
int narrow_linear_bwd(const clid_linear_bwd_args* c, hipStream_t s) {
  BY_DTYPE(c->dtype, {
    Narrow a = narrow_args<T>(c->x, c->ldx, c->w, c->ldw, nullptr, c->rows, c->k, c->n);
    a.dy = c->dy; a.lddy = c->lddy; a.z_in = c->act == CLID_ACT_NONE ? nullptr : c->z; a.act = c->act; a.z_is_y = c->z_is_y;
    a.dx = c->dx; a.part = (float*)c->ws; a.want_w = c->dw != nullptr;
    return narrow_bwd<T, Do::LinearBwd>(a, c->dw, c->db, s);
  });
}
int64_t narrow_ce_bytes(const clid_ce_args* c) {
  const int64_t strips = (c->rows + 31) / 32;
  return up256((strips < kMostBlocks ? strips : kMostBlocks) * 16);
}
int narrow_ce(const clid_ce_args* c, hipStream_t s) {
  int blocks = 0;
  BY_DTYPE(c->dtype, {
    Narrow a = narrow_args<T>(c->x, c->ldx, c->w, c->ldw, c->bias, c->rows, c->k, c->n);
    a.target = c->target; a.ignore = c->ignore_index;
    a.loss_none = c->reduction == CLID_REDUCE_NONE ? c->loss_out : nullptr;
    a.sums = (double*)c->ws;
    blocks = narrow_by_shape<T, Do::Ce>(a, s);
  });
  if (blocks < 0) return blocks;
  hipLaunchKernelGGL(k_narrow_total, dim3(1), dim3(256), 0, s, (const double*)c->ws, blocks, c->reduction, (float*)c->saved, c->loss_out);
  return CLID_OK;
}
int64_t narrow_ce_bwd_bytes(const clid_ce_args* c) { return part_bytes_of(c->rows, c->k, c->n); }
int narrow_ce_bwd(const clid_ce_args* c, hipStream_t s) {
  BY_DTYPE(c->dtype, {
    Narrow a = narrow_args<T>(c->x, c->ldx, c->w, c->ldw, c->bias, c->rows, c->k, c->n);
    a.target = c->target; a.ignore = c->ignore_index; a.reduction = c->reduction; a.g = c->g; a.total = (float*)c->saved;
    a.dx = c->dx; a.part = (float*)c->ws; a.want_w = c->dw != nullptr;
    return narrow_bwd<T, Do::CeBwd>(a, c->dw, c->db, s);
  });
}
int narrow_label(const clid_label_args* c, hipStream_t s) {
  int blocks = 0;
  BY_DTYPE(c->dtype, {
    Narrow a = narrow_args<T>(c->x, c->ldx, c->w, c->ldw, c->bias, c->rows, c->k, c->n);
    a.label = c->label; a.log_prob = c->log_prob;
    blocks = narrow_by_shape<T, Do::Label>(a, s);
  });
  return blocks < 0 ? blocks : CLID_OK;
}

}  // namespace clid_dense
