// The matrix-core product under the dense operators: OUT(m, n) = sum_k P(m, k) Q(n, k), fp32 sums, 16-bit operands.
//
// Operands.  P and Q lie in memory either with k contiguous (rows of a layer's input, a weight) or with k as the row (KS: the
// same matrices seen from the gradients' products); both go through LDS as they lie, and the fragments of a KS operand are
// turned on the way out of LDS (ds_read_b64_tr_b16), so no transposed copy is ever made.
// fp32 operands come as NP = 3 bf16 planes, hi + mid + lo = v exactly (8 bits each, by truncation), 32 columns' hi, their mid, their lo in
// turn, so that a row's copy to LDS is 192 neighbouring bytes and not three times 64 (half a cache line each): six plane products
// (hi hi, hi mid, mid hi, mid mid, hi lo, lo hi) leave out less than 2^-21 of |p q| (mid lo and lo mid: mid is under 2^-7, lo under 2^-15
// of its number; under 2^-24 on average) and run at the bf16 rate, 2.5 PFLOP/s / 6 = 417 TFLOP/s against 157 of the fp32 matrix instructions.
//
// Tiles.  One block computes BM x BN with WM x WN waves, each 32 x 32 x 16 instructions on a (BM / WM) x (BN / WN) part.  Per step
// of BK along k the block copies both tiles from memory straight to LDS (16 bytes a lane, buffer loads whose bounds check turns
// everything outside the matrix into zeros), one step ahead, into the other half of LDS, while the waves multiply.
// LDS rows are dealt out in 16-byte chunks whose place is permuted per row so that the lanes that read together hit different
// banks; the copy writes LDS in lane order, so the permutation is applied to the address each lane loads from.
// The instruction's row operand is Q, its column operand P: a lane then holds one m and, per instruction, four runs of four
// neighbouring n -- stores are 8 or 16 bytes wide and a row's softmax statistics need one exchange between two lanes.
//
// Blocks.  Block ids go round the 8 XCDs in turn; consecutive tiles of one XCD share rows of Q (8 of them, then the next m), so that an
// XCD's 32 CUs work on an 8 x 4 patch of tiles out of their own L2.
//
// Measured: 8192 x 8192 x 8192 bf16 1.01 ms one after the other (1090 TFLOP/s; the matrix pipes are busy for 60 % of the cycles, at a clock that
// the power limit takes from 1.9 to 1.55 GHz), 4096 x 4096 x 4096 fp32 0.66 ms (208 TFLOP/s of fp32 products, 6 x that on the pipes).  The 256 x 256
// tile with 4 waves of 128 x 128 reached 950 to 1100 TFLOP/s, with steps of 32 and four of them in LDS (64-byte rows) 900 to 1150, fp32 with
// steps of 16 0.80 ms.
#pragma once
#include "dense.hpp"

namespace clid_dense {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;

struct Operand {
  const uint16_t* p;
  int64_t ld;  // elements between rows, the planes' included
};

// where column c (a multiple of 8) of a row begins, in elements; plane s is 32 s behind it
template <int NP>
__host__ __device__ __forceinline__ int64_t column(int64_t c) { return NP == 3 ? (c >> 5) * 96 + (c & 31) : c; }

struct Product {
  Operand p, q;
  int64_t m, n, k;      // k (contiguous operands) or the rows' lengths (KS ones) are multiples of 8, by zeros where need be
  const int32_t* live;  // how many of m (or of k, live_k) there are on the device; NULL: all
  int live_k;
  int splits;           // k is cut into so many parts, part s of tile t is block t * splits + s
  int tiles_m, tiles_n, first_m;  // of this launch: its tiles, and the tile rows before them
};

template <bool F16>
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

constexpr uint32_t kOutside = 0x80000000u;  // an offset that every bounds check here refuses: the load returns zeros

// 16 bytes a lane from base + offset (zeros where they end behind `bound`) to lds + 16 lane
__device__ __forceinline__ void copy16(const void* base, uint32_t bound, uint32_t offset, char* lds) {
  auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bound, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
}

// v as three bf16 planes, each the one before's remainder cut to 8 bits: their sum is v.  An infinity or a NaN has it all in the first, whose
// products have sums of their own (k_tile); a value under 2^-133 keeps at least its sign there.
__device__ __forceinline__ void planes(float v, uint16_t (&h)[3]) {
  const uint32_t b = __float_as_uint(v);
  if ((b & 0x7f800000u) == 0x7f800000u) {
    h[0] = (uint16_t)((b >> 16) | ((b & 0x7fffffu) ? 0x40 : 0));
    h[1] = h[2] = 0;
    return;
  }
  const float r1 = v - __uint_as_float(b & 0xffff0000u);
  const uint32_t b1 = __float_as_uint(r1) & 0xffff0000u;
  h[0] = (uint16_t)((b >> 16) | ((b & 0x7fff0000u) == 0 && (b & 0xffffu) ? 1 : 0));
  h[1] = (uint16_t)(b1 >> 16);
  h[2] = (uint16_t)(__float_as_uint(r1 - __uint_as_float(b1)) >> 16);
}

// 4 rows of 16 columns turned: lane i of 16 gives the address of 4 columns of row i / 4 and gets column i of the four rows.  (__restrict__
// puts alias information on the read; without any the compiler waits for every copy to LDS under way before it, also for the next
// step's, which is what arrive() is for.)
__device__ __forceinline__ s16x4 turned(const char* __restrict__ at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
}

// R rows (m or n) x BK of one operand in LDS, all planes
template <int R, int BK, int NP, bool KS, int WAVES>
struct Side {
  static_assert(NP == 1 || BK == 32, "a step of fp32 is a block of planes");
  static constexpr int kBytes = R * BK * 2 * NP;
  static constexpr int kLoads = kBytes / 1024 / WAVES;        // 16-byte loads per lane
  static constexpr int kChunks = (KS ? R : BK) * NP / 8;      // 16-byte chunks of an LDS row
  static_assert(kBytes % (1024 * WAVES) == 0, "whole loads");

  // Where chunk c of LDS row `row` lies.  Reads are free of bank conflicts where 16 lanes hit all of 256 bytes once: one chunk of 16
  // rows, or (KS) 64 bytes of four rows.
  static __device__ __forceinline__ int place(int row, int c) {
    if constexpr (KS) {
      if constexpr (NP == 3) return c ^ ((R == 64 ? row >> 1 & 1 : row & 3) << 2);
      if constexpr (kChunks >= 32) return c ^ ((((row >> 1) & 4) | (row & 3)) << 2);
      if constexpr (kChunks == 16) return c ^ ((row & 3) << 2);
      return c ^ (((row >> 1) & 1) << 2);
    } else {
      if constexpr (NP == 3) return c ^ ((row >> 2) & 3);  // 12 chunks a row: four rows go round the banks three times
      return c ^ ((row / (16 / kChunks)) & (kChunks - 1));
    }
  }

  uint32_t at[kLoads];  // byte offset of this lane's loads within the tile

  // first: the tile's first row (m or n); rows: how many there are
  __device__ __forceinline__ void init(const Operand& o, int64_t first, int64_t rows, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = (i * WAVES + wave) * 64 + lane, row = c / kChunks, chunk = place(row, c % kChunks);
      const int64_t of = KS ? (NP == 3 ? chunk / 12 * 32 : chunk * 8) : row;  // the row of m or n that it belongs to
      at[i] = first + of < rows ? uint32_t(row) * uint32_t(o.ld * 2) + chunk * 16 : kOutside;
    }
  }

  // copies a step of the tile to LDS, all of it below k: nothing to check but at[]
  __device__ __forceinline__ void load(const uint16_t* base, char* lds, int wave) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) copy16(base, 0x7fffffffu, at[i], lds + (i * WAVES + wave) * 1024);
  }
  // the last step of a share that is no multiple of BK: rows (or chunks) from k on are zeros
  __device__ __forceinline__ void load_last(const uint16_t* base, char* lds, int wave, int lane, int left) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = (i * WAVES + wave) * 64 + lane, row = c / kChunks, chunk = place(row, c % kChunks);
      copy16(base, 0x7fffffffu, (KS ? row : (NP == 3 ? chunk % 4 : chunk) * 8) < left ? at[i] : kOutside, lds + (i * WAVES + wave) * 1024);
    }
  }

  // this lane's 8 values of k (16 kk + 8 (lane / 32) ..) of row 32 t + lane % 32, plane s
  static __device__ __forceinline__ s16x8 fragment(const char* lds, int s, int first, int kk, int lane) {
    if constexpr (!KS) {
      const int row = first + (lane & 31), c = s * 4 + 2 * kk + (lane >> 5);
      return *(const s16x8*)(lds + (row * kChunks + place(row, c)) * 16);
    } else {
      // 16 lanes together read 4 rows (k) of 16 columns; lane i of them gets column i of the four rows
      const int i = lane & 15, k = 16 * kk + 8 * (lane >> 5) + (i >> 2), col = first + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
      const int c = NP == 3 ? (first >> 5) * 12 + s * 4 + ((col & 31) >> 3) : col >> 3;
      const s16x4 a = turned(lds + (k * kChunks + place(k, c)) * 16 + (col & 4) * 2);
      const s16x4 b = turned(lds + ((k + 4) * kChunks + place(k + 4, c)) * 16 + (col & 4) * 2);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// LDS of one wave for its sums on their way out, 64 rows at a time, a row 4 floats longer than its columns: neighbouring rows start 4
// banks apart
template <int TM, int TN> constexpr int kRowsLds = (TM > 1 ? 64 : 32) * (32 * TN + 4) * 4;

// LDS in front of the bias: the stages, later the waves' rows
template <int NP, int BM, int BN, int BK, int WM, int WN, int STAGES>
constexpr int tile_lds() {
  const int stages = STAGES * NP * (BM + BN) * BK * 2, rows = WM * WN * kRowsLds<BM / WM / 32, BN / WN / 32>;
  return stages > rows ? stages : rows;
}

// (tile row, tile column) of tile t
__device__ __forceinline__ void place_tile(const Product& g, int64_t block, int64_t blocks, int* tm, int* tn) {
  constexpr int64_t kXcd = 8, kCols = 8;
  int64_t t = block;
  const int64_t whole = blocks / kXcd * kXcd;
  if (t < whole) t = (t % kXcd) * (blocks / kXcd) + t / kXcd;
  const int64_t band = kCols * g.tiles_m, b = t / band, in = t % band;
  const int64_t cols = g.tiles_n - b * kCols < kCols ? g.tiles_n - b * kCols : kCols;
  *tn = (int)(b * kCols + in % cols);
  *tm = (int)(in / cols);
}

template <bool F16, int NP, int BM, int BN, int BK, int WM, int WN, int STAGES, bool PKS, bool QKS, class Epi>
__global__ void __launch_bounds__(64 * WM * WN) k_tile(Product g, Epi epi) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  using SideP = Side<BM, BK, NP, PKS, WAVES>;
  using SideQ = Side<BN, BK, NP, QKS, WAVES>;
  constexpr int kStage = SideP::kBytes + SideQ::kBytes;
  constexpr int kBias = tile_lds<NP, BM, BN, BK, WM, WN, STAGES>();
  extern __shared__ __align__(16) char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn;
  place_tile(g, blockIdx.x / g.splits, gridDim.x / g.splits, &tm, &tn);
  const int split = blockIdx.x % g.splits;
  int64_t rows_m = g.m, rows_k = g.k;
  if (g.live) {
    const int64_t live = *g.live;
    if (g.live_k) rows_k = live < rows_k ? live : rows_k;
    else rows_m = live < rows_m ? live : rows_m;
  }
  const int64_t m0 = (int64_t)(g.first_m + tm) * BM, n0 = (int64_t)tn * BN;
  if (m0 >= rows_m) return;
  const int steps_all = (int)((rows_k + BK - 1) / BK), per = (steps_all + g.splits - 1) / g.splits;
  const int first = split * per, steps = first + per < steps_all ? per : steps_all > first ? steps_all - first : 0;
  const int last = (int)(rows_k - (int64_t)(first + steps - 1) * BK < BK ? rows_k - (int64_t)(first + steps - 1) * BK : BK);  // values of the last step

  // rows of a KS operand are as long as its matrix, padded
  constexpr int64_t kPad = NP == 3 ? 31 : 7;
  const int64_t lim_m = PKS ? (rows_m + kPad) & ~kPad : rows_m, lim_n = QKS ? (g.n + kPad) & ~kPad : g.n;
  SideP sp;
  SideQ sq;
  sp.init(g.p, m0, lim_m, wave, lane);
  sq.init(g.q, n0, lim_n, wave, lane);
  // fp32: hi hi has sums of its own, and the five smaller products theirs, 2^-8 of it: one rounding of the large sum a step and not six
  f32x16 acc[TM][TN], small[NP == 3 ? TM : 1][NP == 3 ? TN : 1];
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[j][i][r] = 0.f;
        if constexpr (NP == 3) small[j][i][r] = 0.f;
      }

  constexpr int kLoads = SideP::kLoads + SideQ::kLoads;  // of a lane and step
  const int64_t p_step = PKS ? BK * g.p.ld : BK * NP, q_step = QKS ? BK * g.q.ld : BK * NP;
  const uint16_t* p_at = g.p.p + (PKS ? column<NP>(m0) : m0 * g.p.ld) + first * p_step;
  const uint16_t* q_at = g.q.p + (QKS ? column<NP>(n0) : n0 * g.q.ld) + first * q_step;
  int loaded = 0;
  auto load = [&]() {  // the next step's
    char* buf = lds + loaded % STAGES * kStage;
    if (loaded + 1 < steps || last == BK) {
      sp.load(p_at, buf, wave);
      sq.load(q_at, buf + SideP::kBytes, wave);
    } else {
      sp.load_last(p_at, buf, wave, lane, last);
      sq.load_last(q_at, buf + SideP::kBytes, wave, lane, last);
    }
    ++loaded;
    p_at += p_step;
    q_at += q_step;
  };
  struct Frags {
    s16x8 p[NP][TM], q[NP][TN];
  };
  auto read = [&](const char* buf, int kk, Frags& f) {
#pragma unroll
    for (int s = 0; s < NP; ++s) {
#pragma unroll
      for (int j = 0; j < TM; ++j) f.p[s][j] = SideP::fragment(buf, s, (wm * TM + j) * 32, kk, lane);
#pragma unroll
      for (int i = 0; i < TN; ++i) f.q[s][i] = SideQ::fragment(buf + SideP::kBytes, s, (wn * TN + i) * 32, kk, lane);
    }
  };
  auto multiply = [&](const Frags& f) {
    if constexpr (NP == 3) {
      constexpr int kP[5] = {0, 2, 1, 0, 1}, kQ[5] = {2, 0, 1, 1, 0};
#pragma unroll
      for (int t = 0; t < 5; ++t)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int i = 0; i < TN; ++i) small[j][i] = mfma<F16>(f.q[kQ[t]][i], f.p[kP[t]][j], small[j][i]);
    }
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int i = 0; i < TN; ++i) acc[j][i] = mfma<F16>(f.q[0][i], f.p[0][j], acc[j][i]);
  };
  // Step s + 1 is there for this wave when nothing but the loads of the steps behind it is under way, and for every wave behind the barrier,
  // where also nobody reads step s any more: its part of LDS is the next load's.
  auto arrive = [&](bool more) {
    if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // The fragments of a product are read while the one before is multiplied, also across the barrier: the matrix pipes have the last
  // product of step s to do while the first fragments of step s + 1 come.
  constexpr int KK = BK / 16;
  static_assert(KK % 2 == 0, "a step's first fragments are f[0]");
  constexpr bool kAcross = STAGES >= 3;         // (two stages: the copy is too late for that)
  constexpr bool kAhead = NP == 1 || kAcross;   // (fp32's large tile has no registers for two: 14 of them would be spilled)
  Frags f[2];
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps) load();
  epi.prepare(n0, lds + kBias);
  if (kAcross && steps > 0) {
    arrive(steps >= STAGES - 1);
    read(lds, 0, f[0]);
  }
  for (int s = 0; s < steps; ++s) {
    const char* buf = lds + s % STAGES * kStage;
    if constexpr (!kAcross) {
      arrive(false);
      read(buf, 0, f[0]);
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      Frags &now = f[kAhead ? kk & 1 : 0], &next = f[(kk + 1) & 1];
      if constexpr (kAhead) {
        if (kk + 1 < KK) {
          read(buf, kk + 1, next);
        } else if (kAcross && s + 1 < steps) {
          arrive(s + STAGES - 1 < steps);
          read(lds + (s + 1) % STAGES * kStage, 0, next);
        }
      } else if (kk) {
        read(buf, kk, now);
      }
      if (kk == 0 && s + STAGES - 1 < steps) load();  // behind the reads that the products wait for
      multiply(now);
      if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);  // without it the compiler moves reads back to their use
    }
  }
  if constexpr (NP == 3) {
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          // an infinity times another operand's plane that is zero made a NaN of the small sum only
          const float v = acc[j][i][r];
          acc[j][i][r] = fabsf(v) <= 3.4028235e38f ? v + small[j][i][r] : v;
        }
  }
  if (Epi::kThroughLds || steps == 0) __syncthreads();  // LDS is the epilogue's; what prepare() left there is seen

  epi.template rows<TM, TN>(acc, m0 + wm * TM * 32, rows_m, n0 + wn * TN * 32, wn * TN * 32, split, lane, lds + kBias, lds + wave * kRowsLds<TM, TN>);
}

}  // namespace clid_dense
