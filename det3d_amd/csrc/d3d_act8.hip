// Rows held in 8 bits, and the weight gradient that reads them (include/d3d.h, d3d_act8_*; arithmetic in d3d_act8.h).
#include "d3d_act8.h"

// ---- hold / restore: one pass over the rows, bound by HBM.  A lane moves one 16-byte vector (or one value of an unaligned row)
// and the lanes of a group agree on its scale by shuffles.  Work items cover whole groups, so the codes behind the last channel
// are written too (as zeros): what reads them later needs no mask.
template <bool BF16, int E, int FMT>
__global__ void __launch_bounds__(256)
    a8_hold_kernel(const void *__restrict__ x, int64_t stride, int64_t n, int c, int pitch, uint8_t *__restrict__ codes,
                   uint8_t *__restrict__ scales) {
  const int per_row = pitch / E;
  const int64_t total = n * per_row;
  // (whole waves stay in the loop: every lane of a group takes part in its shuffles)
  const int64_t rounds = (total + (int64_t)gridDim.x * 256 - 1) / ((int64_t)gridDim.x * 256);
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t i = (k * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    const bool inside = i < total;
    const int64_t row = inside ? i / per_row : 0;
    const int at = inside ? (int)(i - row * per_row) * E : 0;
    float v[E];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = 0.f;
    if (inside && at < c) A8Row<BF16, E>::load(x, row * stride + at, v);
    A8Held<FMT, E, A8_GROUP / E>::store(codes, scales, row, pitch, at, inside, v);
  }
}

template <bool BF16, int E, int FMT>
__global__ void __launch_bounds__(256)
    a8_restore_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t n, int c, int pitch,
                      void *__restrict__ out, int64_t stride) {
  const int per_row = (c + E - 1) / E;
  const int64_t total = n * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int at = (int)(i - row * per_row) * E;
    float v[E];
    A8Held<FMT, E, A8_GROUP / E>::load(codes, scales, row, pitch, at, v);
    A8Row<BF16, E>::store(out, row * stride + at, v);
  }
}

static int a8_check(int64_t n, int c, int dtype, int fmt, const char *who) {
  D3D_REQUIRE(dtype == D3D_F32 || dtype == D3D_BF16, "%s: dtype %d", who, dtype);
  D3D_REQUIRE(fmt == D3D_ACT8_INT8 || fmt == D3D_ACT8_E4M3, "%s: format %d", who, fmt);
  D3D_REQUIRE(n >= 0 && c >= 1 && c <= (1 << 20), "%s: %lld rows of %d channels", who, (long long)n, c);
  return D3D_OK;
}
static unsigned a8_grid(int64_t items) {
  const int64_t nb = (items + 255) / 256;
  return (unsigned)(nb < 1 ? 1 : (nb > 4096 ? 4096 : nb));
}

// KERNEL<type, vector width, format> by the row's type and alignment
#define A8_LAUNCH(KERNEL, VEC, ITEMS_E, ...)                                                                             \
  do {                                                                                                                   \
    const dim3 grid(a8_grid(n * ((int64_t)(ITEMS_E) / ((VEC) ? (dtype == D3D_BF16 ? 8 : 4) : 1)))), block(256);          \
    if (dtype == D3D_BF16 && (VEC)) {                                                                                    \
      if (fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((KERNEL<true, 8, D3D_ACT8_INT8>), grid, block, 0, stream, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<true, 8, D3D_ACT8_E4M3>), grid, block, 0, stream, __VA_ARGS__);                    \
    } else if (dtype == D3D_BF16) {                                                                                      \
      if (fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((KERNEL<true, 1, D3D_ACT8_INT8>), grid, block, 0, stream, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<true, 1, D3D_ACT8_E4M3>), grid, block, 0, stream, __VA_ARGS__);                    \
    } else if (VEC) {                                                                                                    \
      if (fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((KERNEL<false, 4, D3D_ACT8_INT8>), grid, block, 0, stream, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<false, 4, D3D_ACT8_E4M3>), grid, block, 0, stream, __VA_ARGS__);                   \
    } else {                                                                                                             \
      if (fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((KERNEL<false, 1, D3D_ACT8_INT8>), grid, block, 0, stream, __VA_ARGS__); \
      else hipLaunchKernelGGL((KERNEL<false, 1, D3D_ACT8_E4M3>), grid, block, 0, stream, __VA_ARGS__);                   \
    }                                                                                                                    \
  } while (0)

extern "C" int d3d_act8_pitch(int c) { return c >= 1 && c <= (1 << 20) ? a8_pitch(c) : 0; }

extern "C" int d3d_act8_hold(const void *x, int64_t x_stride, int64_t n, int c, int dtype, int fmt, uint8_t *codes,
                             uint8_t *scales, d3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int rc = a8_check(n, c, dtype, fmt, "d3d_act8_hold");
  if (rc) return rc;
  if (n == 0) return D3D_OK;
  D3D_REQUIRE(x && codes && scales, "d3d_act8_hold: null pointer");
  D3D_REQUIRE(x_stride >= c, "d3d_act8_hold: rows of %d channels %lld elements apart", c, (long long)x_stride);
  D3D_REQUIRE(((uintptr_t)codes & 15) == 0, "d3d_act8_hold: codes are not aligned to 16 bytes");
  const int pitch = a8_pitch(c);
  const bool vec = a8_vectors(x, x_stride, c, dtype == D3D_BF16 ? 2 : 4);
  A8_LAUNCH(a8_hold_kernel, vec, pitch, x, x_stride, n, c, pitch, codes, scales);
  D3D_LAUNCH_TRY("a8_hold_kernel");
  return D3D_OK;
}

extern "C" int d3d_act8_restore(const uint8_t *codes, const uint8_t *scales, int64_t n, int c, int fmt, int dtype, void *out,
                                int64_t out_stride, d3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int rc = a8_check(n, c, dtype, fmt, "d3d_act8_restore");
  if (rc) return rc;
  if (n == 0) return D3D_OK;
  D3D_REQUIRE(codes && scales && out, "d3d_act8_restore: null pointer");
  D3D_REQUIRE(out_stride >= c, "d3d_act8_restore: rows of %d channels %lld elements apart", c, (long long)out_stride);
  D3D_REQUIRE(((uintptr_t)codes & 15) == 0, "d3d_act8_restore: codes are not aligned to 16 bytes");
  const int pitch = a8_pitch(c);
  const bool vec = a8_vectors(out, out_stride, c, dtype == D3D_BF16 ? 2 : 4);
  A8_LAUNCH(a8_restore_kernel, vec, vec ? c : c, codes, scales, n, c, pitch, out, out_stride);
  D3D_LAUNCH_TRY("a8_restore_kernel");
  return D3D_OK;
}

// ---- weight gradient: dW[k][ci][co] = sum_o x[nbr[k][o]][ci] dy[o][co]
// A thread owns one (ci, co) of a 16 x 16 tile and walks the rows of its split; the splits' sums go to the workspace and are
// added in split order.
template <bool BF16, int FMT>
__global__ void __launch_bounds__(256)
    a8_wgrad_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t n_in, int cin, int pitch,
                    const void *__restrict__ dy, int64_t dy_stride, int64_t n_out, int cout, const int32_t *__restrict__ nbr,
                    int64_t cap, int64_t rows_per_split, float *__restrict__ part, int64_t part_stride) {
  const int tiles_co = (cout + 15) / 16, tiles_ci = (cin + 15) / 16;
  const int co = (blockIdx.x % tiles_co) * 16 + (threadIdx.x & 15);
  const int ci = (blockIdx.x / tiles_co % tiles_ci) * 16 + (threadIdx.x >> 4);
  const int k = blockIdx.x / (tiles_co * tiles_ci);
  if (ci >= cin || co >= cout) return;
  const int64_t first = blockIdx.y * rows_per_split;
  const int64_t last = first + rows_per_split < n_out ? first + rows_per_split : n_out;
  float sum = 0.f;
  for (int64_t o = first; o < last; ++o) {
    const int64_t i = nbr ? nbr[k * cap + o] : o;
    if (i < 0 || i >= n_in) continue;
    float x, g;
    A8Held<FMT, 1, 32>::load(codes, scales, i, pitch, ci, &x);
    A8Row<BF16, 1>::load(dy, o * dy_stride + co, &g);
    sum = fmaf(x, g, sum);
  }
  part[blockIdx.y * part_stride + ((int64_t)k * cin + ci) * cout + co] = sum;
}

__global__ void __launch_bounds__(256)
    a8_fold_kernel(const float *__restrict__ part, int64_t count, int splits, float *__restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int p = 0; p < splits; ++p) s += part[p * count + i];
    out[i] = s;
  }
}

static int a8_wgrad_splits(int64_t n_out, int kvol, int cin, int cout) {
  const int64_t tiles = (int64_t)kvol * ((cin + 15) / 16) * ((cout + 15) / 16);
  int64_t s = 4096 / tiles;
  const int64_t most = (n_out + 63) / 64;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s);
}

extern "C" size_t d3d_act8_wgrad_workspace_bytes(int64_t n_out, int kvol, int cin, int cout, int dtype) {
  if (n_out < 1 || kvol < 1 || cin < 1 || cout < 1 || (dtype != D3D_F32 && dtype != D3D_BF16)) return 0;
  const int splits = a8_wgrad_splits(n_out, kvol, cin, cout);
  return splits > 1 ? (size_t)splits * kvol * cin * cout * sizeof(float) : 0;
}

extern "C" int d3d_act8_wgrad(const uint8_t *codes, const uint8_t *scales, int fmt, int64_t n_in, int cin, const void *dy,
                              int64_t dy_stride, int dtype, int64_t n_out, int cout, const int32_t *nbr, int64_t cap, int kvol,
                              float *dw, void *workspace, size_t workspace_bytes, d3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int rc = a8_check(n_in, cin, dtype, fmt, "d3d_act8_wgrad");
  if (rc) return rc;
  D3D_REQUIRE(n_in >= 1 && n_out >= 1, "d3d_act8_wgrad: n_in=%lld n_out=%lld (empty gradients are the caller's business)",
              (long long)n_in, (long long)n_out);
  D3D_REQUIRE(cout >= 1 && cout <= (1 << 20) && kvol >= 1 && kvol <= 4096, "d3d_act8_wgrad: cout=%d kvol=%d", cout, kvol);
  D3D_REQUIRE((int64_t)kvol * cin * cout < ((int64_t)1 << 31), "d3d_act8_wgrad: a weight of %d x %d x %d", kvol, cin, cout);
  D3D_REQUIRE(n_in < ((int64_t)1 << 31) && n_out < ((int64_t)1 << 31), "d3d_act8_wgrad: %lld / %lld rows", (long long)n_in, (long long)n_out);
  D3D_REQUIRE(codes && scales && dy && dw, "d3d_act8_wgrad: null pointer");
  D3D_REQUIRE(dy_stride >= cout, "d3d_act8_wgrad: rows of %d channels %lld elements apart", cout, (long long)dy_stride);
  D3D_REQUIRE(nbr ? cap >= n_out : (kvol == 1 && n_in == n_out), "d3d_act8_wgrad: cap=%lld kvol=%d n_in=%lld n_out=%lld",
              (long long)cap, kvol, (long long)n_in, (long long)n_out);
  const size_t need = d3d_act8_wgrad_workspace_bytes(n_out, kvol, cin, cout, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return d3d_set_error(D3D_ECAPACITY, "d3d_act8_wgrad: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int splits = a8_wgrad_splits(n_out, kvol, cin, cout), pitch = a8_pitch(cin);
  const int64_t count = (int64_t)kvol * cin * cout, per = (n_out + splits - 1) / splits;
  float *part = splits > 1 ? (float *)workspace : dw;
  const dim3 grid((unsigned)(kvol * ((cin + 15) / 16) * ((cout + 15) / 16)), (unsigned)splits);
#define A8_WG(BF, F) hipLaunchKernelGGL((a8_wgrad_kernel<BF, F>), grid, dim3(256), 0, stream, codes, scales, n_in, cin, pitch, dy, \
                                        dy_stride, n_out, cout, nbr, cap, per, part, count)
  if (dtype == D3D_BF16) { if (fmt == D3D_ACT8_INT8) A8_WG(true, D3D_ACT8_INT8); else A8_WG(true, D3D_ACT8_E4M3); }
  else { if (fmt == D3D_ACT8_INT8) A8_WG(false, D3D_ACT8_INT8); else A8_WG(false, D3D_ACT8_E4M3); }
#undef A8_WG
  D3D_LAUNCH_TRY("a8_wgrad_kernel");
  if (splits > 1) {
    hipLaunchKernelGGL(a8_fold_kernel, dim3(a8_grid(count)), dim3(256), 0, stream, part, count, splits, dw);
    D3D_LAUNCH_TRY("a8_fold_kernel");
  }
  return D3D_OK;
}
