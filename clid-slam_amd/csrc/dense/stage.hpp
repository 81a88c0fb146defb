// Operands made ready for the tiles (tile.hpp): copies with padded rows, bf16 planes of fp32, dz of a layer, column sums, and the
// choice of tile.
#pragma once
#include <atomic>
#include <type_traits>

#include "epi.hpp"

namespace clid_dense {

template <typename T> struct Kind;  // NP: planes a value takes, F16: the matrix instruction
template <> struct Kind<float> { static constexpr int NP = 3; static constexpr bool F16 = false; using E = bf16; };
template <> struct Kind<bf16> { static constexpr int NP = 1; static constexpr bool F16 = false; using E = bf16; };
template <> struct Kind<f16> { static constexpr int NP = 1; static constexpr bool F16 = true; using E = f16; };

inline int64_t up8(int64_t v) { return (v + 7) & ~int64_t(7); }
// columns of a copy that the tiles read: zeros up to a whole chunk, or a whole block of planes
template <typename T> inline int64_t padded(int64_t cols) { return Kind<T>::NP == 3 ? (cols + 31) & ~int64_t(31) : up8(cols); }
constexpr int64_t kLdMost = int64_t(1) << 22;  // a tile's offsets stay under 2^31 bytes

// 8 values as the planes of T at to (aligned to 16 bytes)
template <typename T>
__device__ __forceinline__ void put8(uint16_t* to, const float (&v)[8]) {
  if constexpr (Kind<T>::NP == 1) {
    union { uint4 w; T t[8]; } u;
#pragma unroll
    for (int q = 0; q < 8; ++q) u.t[q] = down<T>(v[q]);
    *(uint4*)to = u.w;
  } else {
    union { uint4 w; uint16_t t[8]; } u[3];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      uint16_t h[3];
      planes(v[q], h);
#pragma unroll
      for (int s = 0; s < 3; ++s) u[s].t[q] = h[s];
    }
#pragma unroll
    for (int s = 0; s < 3; ++s) *(uint4*)(to + s * 32) = u[s].w;
  }
}
// rows of src (in `order`, as many as are live) -> rows of kp values in planes, zeros behind k.  Bound by memory: 32000 x 1024 fp32 (131 MB
// read, 197 written) 50 us.
struct Staging {
  const void* src;
  int64_t ld, rows;
  const int32_t *order, *live;
  char* dst;
  int k, kp, blocks;  // blocks: 0 where the caller's own rows are read
};
// Two operands in one launch, which is 3 us less than two: 333 x 300 -> 200 fp32 layer and gradients 47 -> 42 us, 1999 x 1000 -> 777 layer 46 -> 43.
template <typename T>
__global__ void __launch_bounds__(256) k_stage(Staging a, Staging b) {
  const bool second = (int)blockIdx.x >= a.blocks;
  const Staging& o = second ? b : a;
  const T* src = (const T*)o.src;
  uint16_t* dst = (uint16_t*)o.dst;
  const int32_t* order = o.order;
  const int64_t rows = o.live && *o.live < o.rows ? *o.live : o.rows, ld = o.ld;
  constexpr int NP = Kind<T>::NP;
  const int k = o.k, kp = o.kp, per = kp / 8;
  for (int64_t i = (int64_t)(blockIdx.x - (second ? a.blocks : 0)) * 256 + threadIdx.x; i < rows * per; i += (int64_t)o.blocks * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    float v[8];
    get8(src + (order ? (int64_t)order[r] : r) * ld + c, v, k - c < 8 ? k - c : 8);
    put8<T>(dst + r * kp * NP + column<NP>(c), v);
  }
}

inline dim3 grid_for(int64_t items, int64_t most = 16384) {
  const int64_t b = (items + 255) / 256;
  return dim3((unsigned)(b < 1 ? 1 : b < most ? b : most));
}

// An operand as the tiles read it: the caller's own rows where they are 16-bit, aligned and whole, else a copy in the workspace
template <typename T>
inline bool direct(const void* p, int64_t ld, int k) {
  return Kind<T>::NP == 1 && k % 8 == 0 && ld % 8 == 0 && ld <= kLdMost && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
template <typename T>
inline int64_t stage_bytes(const void* p, int64_t ld, int64_t rows, int k, bool always = false) {
  return direct<T>(p, ld, k) && !always ? 0 : up256(Kind<T>::NP * rows * padded<T>(k) * 2);
}
// what there is to do for one operand (blocks: nothing), and how the tiles read it then
template <typename T>
inline Staging staging(const void* p, int64_t ld, int64_t rows, int k, char* ws, bool always = false, const int32_t* order = nullptr, const int32_t* live = nullptr) {
  const int64_t kp = padded<T>(k);
  return {p, ld, rows, order, live, ws, k, (int)kp, direct<T>(p, ld, k) && !always ? 0 : (int)grid_for(rows * kp / 8).x};
}
template <typename T>
inline Operand staged(const Staging& o) {
  if (o.blocks == 0) return {(const uint16_t*)o.src, o.ld};
  return {(const uint16_t*)o.dst, (int64_t)o.kp * Kind<T>::NP};
}
template <typename T>
inline void stage(const Staging& a, const Staging& b, hipStream_t s) {
  if (a.blocks + b.blocks) hipLaunchKernelGGL(k_stage<T>, dim3(a.blocks + b.blocks), dim3(256), 0, s, a, b);
}

// dz = dy act'(z) -> planes with rows of np values (dst may be NULL: the sums alone), and its column sums over blocks of rows, before any
// rounding -> part[row block][n].  16-bit dz has one rounding here, since the matrix instruction takes both operands in 16 bits: dx and dw are then
// off by 0.00235 where one rounding of the results gives 0.00166 (8192 x 4096 -> 4096 bf16, relative to the norm); in two parts, which would have no
// more than that, both products run twice (762 us -> about 1230).  A block takes 256 columns (8 a thread) and every gridDim.y-th run of 8 rows.  Bound by memory: 8192 x 4096 bf16 (dy, z and
// dz 67 MB each) 47 us, 4.2 TB/s.
template <typename T, typename Z>
__global__ void __launch_bounds__(256) k_dz(const T* dy, int64_t lddy, const Z* z, int64_t rows, int n, int act, uint16_t* dst, int np, float* part) {
  __shared__ float sums[8][256 + 8];
  const int cg = threadIdx.x & 31, rr = threadIdx.x >> 5, c = blockIdx.x * 256 + cg * 8, count = n - c < 8 ? n - c : 8;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < np) {
    const int64_t step = (int64_t)gridDim.y * 8;
    for (int64_t m = (int64_t)blockIdx.y * 8 + rr; m < rows; m += 2 * step) {  // two rows' loads at once
      const bool two = m + step < rows;
      float v[2][8], y[2][8];
      get8(dy + m * lddy + c, v[0], count);
      if (two) get8(dy + (m + step) * lddy + c, v[1], count);
      if (z) {
        get8(z + m * n + c, y[0], count);
        if (two) get8(z + (m + step) * n + c, y[1], count);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (t && !two) break;
        if (z) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[t][q] = q < count ? act_grad(v[t][q], y[t][q], act) : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) sum[q] += v[t][q];
        if (dst) put8<T>(dst + (m + t * step) * np * Kind<T>::NP + column<Kind<T>::NP>(c), v[t]);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int q = 0; q < 8; ++q) sums[rr][cg * 8 + q] = sum[q];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col < n) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) s += sums[r][threadIdx.x];
    part[(int64_t)blockIdx.y * n + col] = s;
  }
}
// Partial column sums joined in their order, `share` of them into out[blockIdx.y][n]; with `live` only those of rows that there are, `per` rows
// each.  64 columns a block, 16 threads a column.
template <typename T>
__global__ void __launch_bounds__(1024) k_colsum_join(const float* part, int blocks, int share, int n, const int32_t* live, int per, const float* alpha, T* out) {
  __shared__ float p[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  if (live) {
    const int64_t there = ((int64_t)*live + per - 1) / per;
    blocks = there < blocks ? (int)there : blocks;
  }
  const int from = blockIdx.y * share, to = from + share < blocks ? from + share : blocks;
  float s = 0.f;
  if (c < n)
#pragma unroll 4
    for (int b = from + g; b < to; b += 16) s += part[(int64_t)b * n + c];
  p[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g || c >= n) return;
  for (int i = 1; i < 16; ++i) s += p[i][threadIdx.x];
  out[(int64_t)blockIdx.y * n + c] = down<T>((alpha ? *alpha : 1.f) * s);
}
inline int row_blocks(int64_t rows, int n) {
  const int64_t cols = (n + 255) / 256, want = 2048 / cols + 1, most = (rows + 15) / 16;
  return (int)(most < want ? most : want);
}

// more than 64 KB of LDS is asked for, once a kernel and device (the flag costs nothing to set again: no lock)
inline int allow_lds(const void* kernel, int bytes) {
  if (bytes <= 65536) return CLID_OK;
  constexpr int kSlots = 1024;
  static std::atomic<uintptr_t> seen[kSlots];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const uintptr_t key = (uintptr_t)kernel * 64 + (uintptr_t)(dev & 63) + 1;
  std::atomic<uintptr_t>& slot = seen[(key >> 6 ^ key >> 16 ^ key) % kSlots];
  if (slot.load() == key) return CLID_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    clid_set_error("dense kernel: %d bytes of LDS refused: %s", bytes, hipGetErrorString(e));
    return CLID_E_HIP;
  }
  slot.store(key);
  return CLID_OK;
}

// n, k <= 64 (narrow.hip; in tiles, 64 -> 64: fp32 98304 rows 51 us against 25, layer and gradients 157 against 69, cross entropy and gradients
// 212 against 70; bf16 35, 103, 153 against 16, 64, 56.  Only 1000 bf16 rows are as quick in tiles: 7 us against 8.  The border
// is what the registers hold, not where both are even: 1048576 rows, cross entropy and gradients in fp16, 64 -> 64 here 314 us, 64 -> 72 in tiles 1316)
inline bool is_narrow(int32_t k, int32_t n) { return k <= 64 && n <= 64; }
int narrow_linear(const clid_linear_args* a, hipStream_t s);
int64_t narrow_linear_bwd_bytes(const clid_linear_bwd_args* a);
int narrow_linear_bwd(const clid_linear_bwd_args* a, hipStream_t s);
int64_t narrow_ce_bytes(const clid_ce_args* a);
int narrow_ce(const clid_ce_args* a, hipStream_t s);
int64_t narrow_ce_bwd_bytes(const clid_ce_args* a);
int narrow_ce_bwd(const clid_ce_args* a, hipStream_t s);
int narrow_label(const clid_label_args* a, hipStream_t s);

// at most 32 rows (few.hip; the instruction's two column blocks.  In tiles, 4096 -> 8192 and 2048 -> 65536: fp32 one row 114 and 426 us against 25
// and 106, 32 rows 118 and 447 against 46 and 138; bf16 one row 26 and 44 against 14 and 45, label 34 and 94 against 27 and 51; bf16 with 32 rows
// is even or behind (26 and 46 against 26 and 59; label 33 and 94 against 37 and 65).  The cross entropy stays here for its fp32 dz also where
// tiles are quicker: bf16 32 rows, with gradients, 113 and 322 us against 158 and 469)
inline bool is_few(int64_t rows) { return rows <= 32; }
int few_linear(const clid_linear_args* a, hipStream_t s);
int64_t few_linear_bwd_bytes(const clid_linear_bwd_args* a);
int few_linear_bwd(const clid_linear_bwd_args* a, hipStream_t s);
int64_t few_label_bytes(const clid_label_args* a);
int few_label(const clid_label_args* a, hipStream_t s);
int64_t few_ce_bytes(const clid_ce_args* a);
int few_ce(const clid_ce_args* a, float4* stat, float* total, hipStream_t s);
int64_t few_ce_bwd_bytes(const clid_ce_args* a);
int few_ce_bwd(const clid_ce_args* a, const float4* stat, const float* total, hipStream_t s);

// ---- tiles --------------------------------------------------------------------------------------------------------------
template <int NP, int SIZE> struct Tile;
template <> struct Tile<1, 2> { static constexpr int BM = 256, BN = 256, BK = 64, WM = 2, WN = 4, STAGES = 2; };
template <> struct Tile<1, 1> { static constexpr int BM = 128, BN = 128, BK = 64, WM = 2, WN = 2, STAGES = 4; };
template <> struct Tile<1, 0> { static constexpr int BM = 64, BN = 64, BK = 64, WM = 2, WN = 2, STAGES = 4; };
template <> struct Tile<3, 2> { static constexpr int BM = 256, BN = 128, BK = 32, WM = 4, WN = 2, STAGES = 2; };
template <> struct Tile<3, 1> { static constexpr int BM = 128, BN = 128, BK = 32, WM = 4, WN = 2, STAGES = 3; };
template <> struct Tile<3, 0> { static constexpr int BM = 64, BN = 64, BK = 32, WM = 2, WN = 2, STAGES = 3; };
template <int NP>
inline void tile_shape(int size, int* bm, int* bn, int* bk) {
  *bm = size == 2 ? Tile<NP, 2>::BM : size == 1 ? Tile<NP, 1>::BM : Tile<NP, 0>::BM;
  *bn = size == 2 ? Tile<NP, 2>::BN : size == 1 ? Tile<NP, 1>::BN : Tile<NP, 0>::BN;
  *bk = size == 2 ? Tile<NP, 2>::BK : size == 1 ? Tile<NP, 1>::BK : Tile<NP, 0>::BK;
}

constexpr int kCus = 256;

// Which tile, and into how many parts k is cut: the cheapest by an estimate of the time.  A CU works through its blocks one
// after the other (rounds of 256 blocks) at a rate that grows with the tile, since a larger tile reads less LDS and memory per
// product; a part costs its sums' trip through memory and back, and a launch.  The rates are about those of 8192 x 2048 x 8192 bf16 (tiles
// 64, 128, 256: 474, 396, 256 us) and 2048 x 1024 x 8192 fp32 (274, 209, 194 us); a cut costs 13 us at 2048 x 1024 x 1024 bf16 in two
// parts (13.3 -> 26.6 us) and gains at 128 x 8192 x 1024 in eight (40 -> 17.7 us).  Nor is it faster than the operands come, every tile's own,
// out of the L2s: 14 TB/s (333 x 50024 x 768 bf16: 112 us in 7 parts of tile 64, 57 in 32 of tile 256).
struct Plan {
  int size, splits;
};
template <int NP>
inline Plan plan(int64_t m, int64_t n, int64_t k, bool may_split) {
  constexpr double rate[3] = {NP == 3 ? 2.6e12 : 2.3e12, NP == 3 ? 3.7e12 : 2.8e12, NP == 3 ? 4.2e12 : 4.6e12};  // plane products' FLOP/s of a CU
  Plan best = {0, 1};
  double least = 1e300;
  for (int size = 0; size <= 2; ++size) {
    int bm, bn, bk;
    tile_shape<NP>(size, &bm, &bn, &bk);
    const int64_t tiles = ((m + bm - 1) / bm) * ((n + bn - 1) / bn), steps = (k + bk - 1) / bk;
    for (int s = 1; s <= (may_split ? 64 : 1) && (s == 1 || s * 4 <= steps); s += s < 8 ? 1 : 8) {
      const double rounds = (double)((tiles * s + kCus - 1) / kCus);
      const double share = (double)((steps + s - 1) / s) * bk;
      double t = rounds * (2.0 * bm * bn * share * (NP == 3 ? 6 : 1) / rate[size] + 1e-6);
      const double traffic = (double)tiles * (bm + bn) * k * 2 * NP / 14e12;
      if (t < traffic) t = traffic;
      if (s > 1) t += 6e-6 + (double)s * m * n * 8 / 4e12;
      if (t < least) {
        least = t;
        best = {size, s};
      }
    }
  }
  return best;
}

template <typename T, int SIZE, bool PKS, bool QKS, class Epi>
inline int launch_one(Product g, const Epi& epi, hipStream_t s) {
  constexpr int NP = Kind<T>::NP;
  using C = Tile<NP, SIZE>;
  g.tiles_n = (int)((g.n + C::BN - 1) / C::BN);
  constexpr int kLds = tile_lds<NP, C::BM, C::BN, C::BK, C::WM, C::WN, C::STAGES>() + C::BN * 4;
  static_assert(kLds <= 160 * 1024, "a block fits a CU");
  auto k = k_tile<Kind<T>::F16, NP, C::BM, C::BN, C::BK, C::WM, C::WN, C::STAGES, PKS, QKS, Epi>;
  const int rc = allow_lds((const void*)k, kLds);
  if (rc != CLID_OK) return rc;
  // as many rows of tiles a launch as 2^32 threads take (one row of them is under 2^29: n < 2^20, at most 64 splits)
  const int64_t tiles_m = (g.m + C::BM - 1) / C::BM, each = (int64_t)g.tiles_n * g.splits, most = ((int64_t(1) << 32) - 1) / (each * 64 * C::WM * C::WN);
  for (int64_t t = 0; t < tiles_m; t += most) {
    g.first_m = (int)t;
    g.tiles_m = (int)(tiles_m - t < most ? tiles_m - t : most);
    hipLaunchKernelGGL(k, dim3((unsigned)(g.tiles_m * each)), dim3(64 * C::WM * C::WN), kLds, s, g, epi);
  }
  return CLID_OK;
}

template <typename T, bool PKS, bool QKS, class Out>
inline int launch_rows(const Product& g, int size, const Out& o, hipStream_t s) {
  constexpr int NP = Kind<T>::NP;
  if (size == 2) return launch_one<T, 2, PKS, QKS>(g, EpiRows<Out, Tile<NP, 2>::BN>{o, g.n}, s);
  if (size == 1) return launch_one<T, 1, PKS, QKS>(g, EpiRows<Out, Tile<NP, 1>::BN>{o, g.n}, s);
  return launch_one<T, 0, PKS, QKS>(g, EpiRows<Out, Tile<NP, 0>::BN>{o, g.n}, s);
}
template <typename T, bool PKS, bool QKS, class Out>
inline int launch_out(Product g, const Plan& p, const Out& o, char* part, hipStream_t s) {
  g.splits = p.splits;
  if (p.splits == 1) return launch_rows<T, PKS, QKS>(g, p.size, o, s);
  const int64_t n8 = up8(g.n);
  const int rc = launch_rows<T, PKS, QKS>(g, p.size, PartOut{nullptr, (float*)part, g.m, n8}, s);
  if (rc != CLID_OK) return rc;
  const int32_t* live = g.live_k ? nullptr : g.live;
  if (p.splits > 8) hipLaunchKernelGGL((k_join<T, Out, 8>), grid_for(g.m * n8), dim3(256), 0, s, (const float*)part, p.splits, g.m, n8, live, o);
  else hipLaunchKernelGGL((k_join<T, Out, 1>), grid_for(g.m * n8 / 8), dim3(256), 0, s, (const float*)part, p.splits, g.m, n8, live, o);
  return CLID_OK;
}
inline int64_t part_bytes(const Plan& p, int64_t m, int64_t n) { return p.splits > 1 ? up256(p.splits * m * up8(n) * 4) : 0; }

// the workspace handed out front to back; sizes and pointers come from one walk, so they cannot differ
struct Ws {
  char* base;
  int64_t used = 0;
  explicit Ws(void* p) : base((char*)p) {}
  char* take(int64_t bytes) {
    char* at = base ? base + used : nullptr;
    used += up256(bytes);
    return at;
  }
};

inline int bad(const char* what, const char* why) {
  clid_set_error("%s: %s", what, why);
  return CLID_E_ARG;
}
// a workspace of `need` bytes as the header asks for it
inline bool ws_ok(const void* ws, int64_t bytes, int64_t need) { return need == 0 || (ws && bytes >= need && (reinterpret_cast<uintptr_t>(ws) & 255) == 0); }
inline bool dtype_ok(int d) { return d == CLID_F32 || d == CLID_BF16 || d == CLID_F16; }

}  // namespace clid_dense

#define BY_DTYPE(dtype, ...)                                       \
  do {                                                             \
    if ((dtype) == CLID_F32) { using T = float; __VA_ARGS__ }      \
    else if ((dtype) == CLID_BF16) { using T = clid_dense::bf16; __VA_ARGS__ } \
    else { using T = clid_dense::f16; __VA_ARGS__ }                \
  } while (0)
