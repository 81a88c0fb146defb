// A layer: y = act(x w^T + bias) + residual, and its gradients (include/clid_dense.h).
#include "stage.hpp"

using namespace clid_dense;

namespace {

template <typename T>
struct Fwd {
  Plan p;
  char *x, *w, *part;
  int64_t bytes;
  explicit Fwd(const clid_linear_args* a) {
    Ws ws(a->ws);
    // both copies or neither where k is odd: their rows are padded alike
    x = ws.take(stage_bytes<T>(a->x, a->ldx, a->rows, a->k));
    w = ws.take(stage_bytes<T>(a->w, a->ldw, a->n, a->k));
    p = plan<Kind<T>::NP>(a->rows, a->n, a->k, true);
    part = ws.take(part_bytes(p, a->rows, a->n));
    bytes = ws.used;
  }
};

template <typename T>
int fwd(const clid_linear_args* a, hipStream_t s) {
  const Fwd<T> f(a);
  const Staging x = staging<T>(a->x, a->ldx, a->rows, a->k, f.x), w = staging<T>(a->w, a->ldw, a->n, a->k, f.w);
  stage<T>(x, w, s);
  Product g = {staged<T>(x), staged<T>(w), a->rows, a->n, up8(a->k), nullptr, 0, 1, 0, 0};
  LinearOut<T> o = {(const T*)a->bias, (const T*)a->residual, (T*)a->y, (typename KeptZ<T>::Z*)a->z_out, a->ldr, a->n, a->act};
  return launch_out<T, false, false>(g, f.p, o, f.part, s);
}

template <typename T>
struct Bwd {
  bool own_dz;  // dz is not dy itself
  int blocks;
  Plan px, pw;
  char *dz, *w, *x, *sums, *part;
  int64_t bytes;
  explicit Bwd(const clid_linear_bwd_args* a) {
    Ws ws(a->ws);
    own_dz = (a->dx || a->dw) && (a->act != CLID_ACT_NONE || !direct<T>(a->dy, a->lddy, a->n));
    dz = ws.take(own_dz ? Kind<T>::NP * a->rows * padded<T>(a->n) * 2 : 0);
    w = ws.take(a->dx ? stage_bytes<T>(a->w, a->ldw, a->n, a->k) : 0);
    x = ws.take(a->dw ? stage_bytes<T>(a->x, a->ldx, a->rows, a->k) : 0);
    blocks = row_blocks(a->rows, a->n);
    sums = ws.take(a->db ? (int64_t)blocks * a->n * 4 : 0);
    px = plan<Kind<T>::NP>(a->rows, a->k, a->n, true);
    pw = plan<Kind<T>::NP>(a->n, a->k, a->rows, true);
    const int64_t bx = a->dx ? part_bytes(px, a->rows, a->k) : 0, bw = a->dw ? part_bytes(pw, a->n, a->k) : 0;
    part = ws.take(bx > bw ? bx : bw);
    bytes = ws.used;
  }
};

template <typename T>
int bwd(const clid_linear_bwd_args* a, hipStream_t s) {
  const Bwd<T> f(a);
  const int np = (int)padded<T>(a->n);
  Operand dz = {(const uint16_t*)a->dy, a->lddy};
  if (f.own_dz) dz = {(const uint16_t*)f.dz, np * Kind<T>::NP};
  if (f.own_dz || a->db) {
    const auto launch = [&](auto* z) {
      using Z = std::remove_const_t<std::remove_pointer_t<decltype(z)>>;
      hipLaunchKernelGGL((k_dz<T, Z>), dim3((np + 255) / 256, f.blocks), dim3(256), 0, s, (const T*)a->dy, a->lddy, a->act == CLID_ACT_NONE ? nullptr : z, a->rows, a->n,
                         a->act, f.own_dz ? (uint16_t*)f.dz : nullptr, np, a->db ? (float*)f.sums : nullptr);
    };
    if (a->z_is_y) launch((const T*)a->z);
    else launch((const typename KeptZ<T>::Z*)a->z);
    if (a->db)
      hipLaunchKernelGGL(k_colsum_join<T>, dim3((a->n + 63) / 64), dim3(1024), 0, s, (const float*)f.sums, f.blocks, f.blocks, a->n,
                         (const int32_t*)nullptr, 1, (const float*)nullptr, (T*)a->db);
  }
  Staging x = staging<T>(a->x, a->ldx, a->rows, a->k, f.x), w = staging<T>(a->w, a->ldw, a->n, a->k, f.w);
  if (!a->dw) x.blocks = 0;
  if (!a->dx) w.blocks = 0;
  stage<T>(x, w, s);
  if (a->dx) {
    Product g = {dz, staged<T>(w), a->rows, a->k, a->n, nullptr, 0, 1, 0, 0};
    const int rc = launch_out<T, false, true>(g, f.px, StoreOut<T>{nullptr, (T*)a->dx, nullptr, nullptr, nullptr, a->k}, f.part, s);
    if (rc != CLID_OK) return rc;
  }
  if (a->dw) {
    Product g = {dz, staged<T>(x), a->n, a->k, a->rows, nullptr, 0, 1, 0, 0};
    return launch_out<T, true, true>(g, f.pw, StoreOut<T>{nullptr, (T*)a->dw, nullptr, nullptr, nullptr, a->k}, f.part, s);
  }
  return CLID_OK;
}

bool args_ok(const clid_linear_args* a) {
  return a && sizes_ok(a->rows, a->k, a->n) && dtype_ok(a->dtype) && a->act >= 0 && a->act <= CLID_ACT_SILU;
}
bool args_ok(const clid_linear_bwd_args* a) {
  return a && sizes_ok(a->rows, a->k, a->n) && dtype_ok(a->dtype) && a->act >= 0 && a->act <= CLID_ACT_SILU;
}

}  // namespace

extern "C" int64_t clid_linear_workspace(const clid_linear_args* a) {
  if (!args_ok(a)) return bad("clid_linear_workspace", "bad argument");
  if (is_narrow(a->k, a->n) || is_few(a->rows)) return 0;
  BY_DTYPE(a->dtype, return Fwd<T>(a).bytes;);
}
extern "C" int clid_linear_fwd(const clid_linear_args* a, void* stream) {
  const char* me = "clid_linear_fwd";
  if (!args_ok(a)) return bad(me, "bad argument");
  if (a->rows == 0) return CLID_OK;
  if (!a->x || !a->w || !a->y || a->ldx < a->k || a->ldw < a->k || (a->residual && a->ldr < a->n)) return bad(me, "bad pointer or row stride");
  const int64_t need = clid_linear_workspace(a);
  if (!ws_ok(a->ws, a->ws_bytes, need)) return bad(me, "workspace too small or not aligned to 256 bytes");
  int rc = CLID_OK;
  if (is_narrow(a->k, a->n)) rc = narrow_linear(a, (hipStream_t)stream);
  else if (is_few(a->rows)) rc = few_linear(a, (hipStream_t)stream);
  else BY_DTYPE(a->dtype, rc = fwd<T>(a, (hipStream_t)stream););
  if (rc != CLID_OK) return rc;
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}

extern "C" int64_t clid_linear_bwd_workspace(const clid_linear_bwd_args* a) {
  if (!args_ok(a)) return bad("clid_linear_bwd_workspace", "bad argument");
  if (is_narrow(a->k, a->n)) return narrow_linear_bwd_bytes(a);
  if (a->dtype == CLID_F32 && is_few(a->rows) && a->rows) return few_linear_bwd_bytes(a);
  BY_DTYPE(a->dtype, return Bwd<T>(a).bytes;);
}
extern "C" int clid_linear_bwd(const clid_linear_bwd_args* a, void* stream) {
  const char* me = "clid_linear_bwd";
  if (!args_ok(a)) return bad(me, "bad argument");
  if (a->rows == 0) return bad(me, "no rows");
  if (!a->x || !a->w || !a->dy || a->ldx < a->k || a->ldw < a->k || a->lddy < a->n || (!a->z && a->act != CLID_ACT_NONE)) return bad(me, "bad pointer or row stride");
  const int64_t need = clid_linear_bwd_workspace(a);
  if (!ws_ok(a->ws, a->ws_bytes, need)) return bad(me, "workspace too small or not aligned to 256 bytes");
  int rc = CLID_OK;
  if (is_narrow(a->k, a->n)) rc = narrow_linear_bwd(a, (hipStream_t)stream);
  else if (a->dtype == CLID_F32 && is_few(a->rows)) rc = few_linear_bwd(a, (hipStream_t)stream);
  else BY_DTYPE(a->dtype, rc = bwd<T>(a, (hipStream_t)stream););
  if (rc != CLID_OK) return rc;
  DENSE_CHECK_LAUNCH(me);
  return CLID_OK;
}
