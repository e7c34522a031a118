// Rows held in 8 bits, and the weight gradient that reads them (include/d3d.h, d3d_act8_*; arithmetic in d3d_act8.h).
#include "d3d_act8.h"

// ---- hold / restore: one pass over the rows, bound by HBM.  A lane moves one vector of 16 bytes and the lanes of a group agree
// on its scale in registers.  Work items cover whole groups, so the codes behind the last channel are written too (as zeros):
// what reads them later needs no mask.  [140800, 128] f32: hold 18.7 us (91 MB, 4.8 TB/s, as a large copy), restore 14.9 us (6.1 TB/s,
// the codes still lie in the caches).
template <bool BF16, int FMT, bool ANY>
__global__ void __launch_bounds__(256)
    a8_hold_kernel(const void *__restrict__ x, int64_t stride, int64_t n, int c, int pitch, uint8_t *__restrict__ codes,
                   uint8_t *__restrict__ scales) {
  constexpr int E = BF16 ? 8 : 4, EB = BF16 ? 2 : 4;
  using Row = A8Row<BF16, E>;
  const int per_row = pitch / E;
  const int64_t total = n * per_row;
  // (whole waves stay in the loop: every lane of a group takes part in its exchanges)
  const int64_t rounds = (total + (int64_t)gridDim.x * 256 - 1) / ((int64_t)gridDim.x * 256);
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t i = (k * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    const bool inside = i < total;
    const int64_t row = inside ? i / per_row : 0;
    const int at = inside ? (int)(i - row * per_row) * E : 0;
    float v[E];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = 0.f;
    if (inside && at < c) Row::template open<ANY>(Row::template get<ANY>((const char *)x + row * stride * EB, at, c), at, c, v);
    A8Held<FMT, E, A8_GROUP / E>::store(codes, scales, row, pitch, at, inside, v);
  }
}

template <bool BF16, int FMT, bool ANY>
__global__ void __launch_bounds__(256)
    a8_restore_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t n, int c, int pitch,
                      void *__restrict__ out, int64_t stride) {
  constexpr int E = BF16 ? 8 : 4, EB = BF16 ? 2 : 4;
  const int per_row = (c + E - 1) / E;
  const int64_t total = n * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int at = (int)(i - row * per_row) * E;
    float v[E];
    A8Held<FMT, E, A8_GROUP / E>::load(codes, scales, row, pitch, at, v);
    A8Row<BF16, E>::template put<ANY>((char *)out + row * stride * EB, at, c, v);
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

// KERNEL<type, format, any alignment and width>
#define A8_LAUNCH(KERNEL, ANY, ITEMS, ...)                                                                                          \
  do {                                                                                                                              \
    const dim3 grid(a8_grid(ITEMS)), block(256);                                                                                    \
    if (dtype == D3D_BF16 && fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((KERNEL<true, D3D_ACT8_INT8, ANY>), grid, block, 0, stream, __VA_ARGS__); \
    else if (dtype == D3D_BF16) hipLaunchKernelGGL((KERNEL<true, D3D_ACT8_E4M3, ANY>), grid, block, 0, stream, __VA_ARGS__);        \
    else if (fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((KERNEL<false, D3D_ACT8_INT8, ANY>), grid, block, 0, stream, __VA_ARGS__);    \
    else hipLaunchKernelGGL((KERNEL<false, D3D_ACT8_E4M3, ANY>), grid, block, 0, stream, __VA_ARGS__);                              \
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
  const int64_t items = n * (pitch / (dtype == D3D_BF16 ? 8 : 4));
  if (a8_vectors(x, x_stride, c, dtype == D3D_BF16 ? 2 : 4)) A8_LAUNCH(a8_hold_kernel, false, items, x, x_stride, n, c, pitch, codes, scales);
  else A8_LAUNCH(a8_hold_kernel, true, items, x, x_stride, n, c, pitch, codes, scales);
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
  const int e = dtype == D3D_BF16 ? 8 : 4;
  const int64_t items = n * ((c + e - 1) / e);
  if (a8_vectors(out, out_stride, c, dtype == D3D_BF16 ? 2 : 4)) A8_LAUNCH(a8_restore_kernel, false, items, codes, scales, n, c, pitch, out, out_stride);
  else A8_LAUNCH(a8_restore_kernel, true, items, codes, scales, n, c, pitch, out, out_stride);
  D3D_LAUNCH_TRY("a8_restore_kernel");
  return D3D_OK;
}

// ---- weight gradient: dW[k][ci][co] = sum_o x[nbr[k][o]][ci] dy[o][co]
//
// A matrix product whose long axis, the rows o, is the outer one of both operands.  Bound by the matrix pipe and by the vector work
// that restores the codes and splits dy, which overlap in part (without the one or the other 46 to 50 us of 57).  65021 sites, 27
// offsets, 64 -> 64 channels, f32: 54 us, 800 TFLOP/s of bf16 products with the absent neighbours' zeros (every second entry);
// [16384, 1024] x [16384, 1024] bf16: 44 us, 780 TFLOP/s, and 11 us to fold the row ranges; 80003 sites, 16 -> 16 bf16: 20 us, bound by
// the gathers: a CU is busy for 38 thousand cycles, the cache is accessed in 21 of them, vector work issues in 9, the waves wait in half.
//
// The (k, ci) axis is flattened (ci padded to 8) and cut into units of 64 columns, so narrow layers fill a unit with several
// offsets.  A block of 8 waves owns KG units x TN columns of dy and a range of rows, 64 rows (a chunk) at a time:
//   * dy's chunk goes through LDS once, as P bf16 planes (f32: three, hi + mid + lo = all 24 bits; restored values are exact in
//     bf16, so the products are exact to f32 either way), and stays in registers as the MFMA's B operand for all KG units;
//   * a unit's 64 x 64 codes are one 8-byte gather a thread, requested a whole chunk (KG units) ahead, its table entry a chunk
//     further; restored to bf16 on the way into LDS (UB units at a time, double buffered, one barrier each);
//   * both operands become MFMA fragments, rows as k, through the transposing read ds_read_b64_tr_b16.
// Wave (wci, wco, wk): 32 of the unit's columns, 32 NB of dy's, every WK-th part of the chunk's rows; the wk parts are added in
// the block, the row ranges through the workspace in their order.
typedef __attribute__((ext_vector_type(4))) short a8_s16x4;
typedef __attribute__((ext_vector_type(8))) short a8_s16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 a8_bf16x8;
typedef __attribute__((ext_vector_type(16))) float a8_f32x16;

#define WG8_ROWS 64
// the schedule of a phase: the fragments' LDS reads, then up to six vector instructions behind each MFMA
#define WG8_INTERLEAVE                                              \
  if (ph == 0) __builtin_amdgcn_sched_group_barrier(0x100, 2 * UB * KS + 2 * KS * NB * P, 0); \
  else __builtin_amdgcn_sched_group_barrier(0x100, 2 * UB * KS, 0); \
  _Pragma("unroll") for (int m = 0; m < UB * KS * NB * P; ++m) {    \
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);              \
    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);              \
  }

struct Wg8Args {
  const uint8_t *codes, *scales;
  const void *dy;
  const int32_t *nbr;
  float *out;  // [splits][kvol][cin][cout], or dw itself
  int64_t dy_stride, cap, count;
  uint32_t n_in, tab_bytes;
  int n_out, cin, cinp, pitch, cout, cols, units, groups, cotiles, chunks, per_split;
};

template <int FMT> __device__ __forceinline__ uint4 wg8_restore(uint2 w, uint32_t b) {
  // 8 codes to bf16: exact
  const float s = a8_up(b);
  if constexpr (FMT == D3D_ACT8_INT8) {
    // a signed byte's conversion is one instruction, scaling another (exact); the upper halves of the f32 values are their bf16
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = __float_as_uint((float)((int)(w.x << (24 - 8 * j)) >> 24) * s);
      v[4 + j] = __float_as_uint((float)((int)(w.y << (24 - 8 * j)) >> 24) * s);
    }
    return make_uint4(__builtin_amdgcn_perm(v[1], v[0], 0x07060302u), __builtin_amdgcn_perm(v[3], v[2], 0x07060302u),
                      __builtin_amdgcn_perm(v[5], v[4], 0x07060302u), __builtin_amdgcn_perm(v[7], v[6], 0x07060302u));
  } else {
    // two codes and the scale's exponent to a pair of bf16 in one instruction
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.x, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.x, s, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.y, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.y, s, true)));
  }
}

// (a function: a conditional between two array elements would choose between their addresses, and put the array in memory)
__device__ __forceinline__ uint32_t wg8_pick(int c, uint32_t a, uint32_t b) { return c ? a : b; }

// byte of 16-byte slot `slot` in row r of a [rows][W columns] bf16 tile.  The slots of a row are permuted so that the four rows
// of a transposing read (64 bytes each) lie in different banks: 128-byte rows alternate halves every second row, wider ones
// rotate quarters of 256 bytes
template <int W> __device__ __forceinline__ uint32_t wg8_slot(int r, int slot) {
  if constexpr (W == 64) slot ^= ((r >> 1) & 1) << 2;
  if constexpr (W >= 128) slot ^= (r & 3) << 2;
  return (uint32_t)(r * (W * 2) + slot * 16);
}

// fragment of mfma_f32_32x32x16_bf16: columns [col, col + 32), rows [row, row + 16) of such a tile; lane l holds column l % 32,
// rows 8 (l / 32) + 0 .. 7
template <int W> __device__ __forceinline__ a8_bf16x8 wg8_fragment(const unsigned char *tile, int row, int col) {
  const int lane = threadIdx.x & 63, i16 = lane & 15;
  const int r = row + ((lane >> 5) << 3) + (i16 >> 2);
  const int c = col + (((lane >> 4) & 1) << 4) + ((i16 & 3) << 2);
  typedef __attribute__((address_space(3))) a8_s16x4 lds_s16x4;
  const unsigned char *p = tile + wg8_slot<W>(r, c >> 3) + (c & 7) * 2;  // (row r + 4 has the same permutation)
  const a8_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
  const a8_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * W * 2));
  const a8_s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(a8_bf16x8, v);
}

template <int FMT, int P, int WCO, int WK, int NB, int KG, int UB, bool TABLE, int EDGE>
__global__ void __launch_bounds__(512, 2) a8_wgrad_kernel(Wg8Args p) {
  constexpr int TN = WCO * NB * 32, KS = WG8_ROWS / WK / 16;
  constexpr int VPT = TN >= 64 ? TN / 64 : 1;  // vectors of 8 columns of dy a thread stages
  constexpr int ABYTES = WG8_ROWS * 128, DBYTES = WG8_ROWS * TN * 2;
  constexpr int RBYTES = (WK - 1) * 2 * WCO * 4096;
  constexpr int SMEM = 2 * UB * ABYTES + 2 * P * DBYTES > RBYTES ? 2 * UB * ABYTES + 2 * P * DBYTES : RBYTES;
  __shared__ __attribute__((aligned(16))) unsigned char smem[SMEM];
  unsigned char *const sa = smem, *const sd = smem + 2 * UB * ABYTES;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wci = wave & 1, wco = (wave >> 1) % WCO, wk = (wave >> 1) / WCO;
  // blocks of one row range next to each other on one XCD: they read the same rows of dy and the same codes
  int logical;
  {
    const int nb = (int)gridDim.x, q = nb >> 3, r = nb & 7, xcd = (int)blockIdx.x & 7, idx = (int)blockIdx.x >> 3;
    logical = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  }
  const int cot = logical % p.cotiles, group = logical / p.cotiles % p.groups, split = logical / (p.cotiles * p.groups);
  const int co0 = cot * TN, unit0 = group * KG;
  const int nu = p.units - unit0 < KG ? p.units - unit0 : KG;
  const int chunk0 = split * p.per_split;
  const int chunks = p.chunks - chunk0 < p.per_split ? p.chunks - chunk0 : p.per_split;

  // Staging.  A thread owns one row of the chunk and 8 columns of each unit.  Loads stay in flight only while nothing touches
  // their registers: no select behind them, no branch around them.  What is absent (a row or a column behind the last, a table
  // entry out of range) reads beyond the buffer, which gives zeros: the scale 0 makes the row add nothing, whatever dy has there.
  // The range check takes in the vector offset alone: everything that moves is part of it, and the scalar offset is 0.
  // Offsets are 32 bits: the table and the codes behind one stay below 2^31 bytes and 2^24 rows (checked on the host); without a
  // table the base moves with the chunk.
  const int srow = tid >> 3, sseg = tid & 7;
  const int rows_here = p.n_out - chunk0 * WG8_ROWS;  // from the block's first row to the last
  const int my_chunks = srow < rows_here ? min((rows_here - srow + WG8_ROWS - 1) / WG8_ROWS, chunks) : 0;
  uint32_t col_off[KG], tab_off[TABLE ? KG : 1];
  int lim[KG];  // chunks in which this thread has something of the unit
#pragma unroll
  for (int u = 0; u < KG; ++u) {
    const int col = (unit0 + u) * 64 + sseg * 8;
    const bool in = u < nu && col < p.cols;
    const int k = TABLE && in ? col / p.cinp : 0, ci = in ? col - k * p.cinp : 0;
    lim[u] = in ? my_chunks : 0;
    col_off[u] = TABLE ? (uint32_t)ci : (uint32_t)(srow * p.pitch + ci);
    if constexpr (TABLE) tab_off[u] = ((uint32_t)k * (uint32_t)p.cap + (uint32_t)(chunk0 * WG8_ROWS + srow)) * 4u;
  }
  int32_t idx[TABLE ? KG : 1];
  uint2 code[KG];
  uint32_t sc[KG];
  const __amdgpu_buffer_rsrc_t tab_rs = __builtin_amdgcn_make_buffer_rsrc((void *)p.nbr, 0, TABLE ? p.tab_bytes : 0, 0x00020000);
  // of the next chunk, as often as it is called: up to two chunks behind the last.  Rows behind the last read entries of other
  // offsets, which load_code drops, and behind the table's end zeros: an offset is below its 2^31 bytes and four chunks
  auto load_idx = [&](int u) {
    if constexpr (TABLE) {
      idx[u] = __builtin_amdgcn_raw_buffer_load_b32(tab_rs, (int)tab_off[u], 0, 0);
      tab_off[u] += WG8_ROWS * 4u;
    }
  };
  auto load_code = [&](int u, int chunk) {
    bool in = chunk < lim[u];
    uint32_t off = col_off[u];
    if constexpr (TABLE) {
      in = in & ((uint32_t)idx[u] < p.n_in);
      off += __umul24((uint32_t)idx[u], (uint32_t)p.pitch);
    }
    off = in ? off : D3D_OOB_OFFSET;
    const int64_t base = TABLE ? 0 : (int64_t)(chunk0 + chunk) * WG8_ROWS * p.pitch;
    code[u] = d3d_buffer_load8(d3d_make_rsrc(p.codes + base), off);
    // (a row of codes is a whole number of groups: group = off / 32; the absent offset / 32 lies behind 2^26 groups)
    sc[u] = __builtin_amdgcn_raw_buffer_load_b8(__builtin_amdgcn_make_buffer_rsrc((void *)(p.scales + (base >> 5)), 0, 1 << 26, 0x00020000), (int)(off >> 5), 0, 0);
  };

  // dy: this thread's vectors of 8 columns of the chunk, as they come; a row behind the last is the last one again (its partner
  // in x is zero).  EDGE: 0 = the width is a multiple of 8; 1 = it is not: the vector that passes a row's end is the row's last 8
  // values, shifted into place on their way to LDS; 2 = rows shorter than a vector: value by value, the last one again behind it
  // (what stands in columns behind the last is multiplied and not stored)
  constexpr int DW = P == 3 || EDGE == 2 ? 8 : 4, EB = P == 3 ? 4 : 2;  // words of a vector, bytes of a value
  uint32_t dyr[VPT][DW];
  const char *dyp[VPT];
  int dy_chunk = 0;
  const int dy_co = co0 + tid % (TN / 8) * 8, dy_at = EDGE == 2 ? dy_co : (EDGE == 1 ? min(dy_co, p.cout - 8) : (dy_co < p.cout ? dy_co : 0));
  const int dy_shift = min(dy_co - dy_at, 8);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = tid + 512 * v, r = i / (TN / 8);
    const int row = r < rows_here ? r : rows_here - 1;
    dyp[v] = (const char *)p.dy + ((int64_t)(chunk0 * WG8_ROWS + row) * p.dy_stride + dy_at) * EB;
  }
  auto load_dy = [&]() {  // of the next chunk, as often as it is called
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      if constexpr (EDGE == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const char *src = dyp[v] + (dy_co + j < p.cout ? j : p.cout - 1 - dy_co) * EB;
          if constexpr (P == 3) dyr[v][j] = *(const uint32_t *)src;
          else dyr[v][j] = *(const uint16_t *)src;
        }
      } else {
        const uint4 x = a8_get<uint4>(dyp[v]);
        dyr[v][0] = x.x; dyr[v][1] = x.y; dyr[v][2] = x.z; dyr[v][3] = x.w;
        if constexpr (P == 3) {
          const uint4 y = a8_get<uint4>(dyp[v] + 16);
          dyr[v][4] = y.x; dyr[v][5] = y.y; dyr[v][6] = y.z; dyr[v][7] = y.w;
        }
      }
    }
    ++dy_chunk;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {  // on to the next row, while there is one
      const int r = (tid + 512 * v) / (TN / 8);
      if (dy_chunk * WG8_ROWS + r < rows_here) dyp[v] += (int64_t)WG8_ROWS * p.dy_stride * EB;
    }
  };
  auto write_dy = [&](int buf) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int i = tid + 512 * v, r = i / (TN / 8), cv = i % (TN / 8);
      if (TN < 64 && r >= WG8_ROWS) continue;
      const uint32_t at = wg8_slot<TN>(r, cv);
      uint32_t w[P][4];
      if constexpr (EDGE == 1 && P == 3) {
#pragma unroll
        for (int m = 1; m <= 8; m <<= 1)
#pragma unroll
          for (int j = 0; j < 8; ++j) dyr[v][j] = wg8_pick(dy_shift & m, j + m < 8 ? dyr[v][j + m < 8 ? j + m : 0] : 0u, dyr[v][j]);
      } else if constexpr (EDGE == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          dyr[v][j] = wg8_pick(dy_shift & 1, __builtin_amdgcn_alignbit(j < 3 ? dyr[v][j < 3 ? j + 1 : 0] : 0u, dyr[v][j], 16), dyr[v][j]);
#pragma unroll
        for (int m = 1; m <= 4; m <<= 1)
#pragma unroll
          for (int j = 0; j < 4; ++j) dyr[v][j] = wg8_pick(dy_shift & 2 * m, j + m < 4 ? dyr[v][j + m < 4 ? j + m : 0] : 0u, dyr[v][j]);
      }
      if constexpr (P == 3) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a = __uint_as_float(dyr[v][2 * j]), b = __uint_as_float(dyr[v][2 * j + 1]);
#pragma unroll
          for (int q = 0; q < 3; ++q) {  // bf16 of what is left, and what that leaves (exact)
            w[q][j] = a8_pack_bf16(a, b);
            a -= __uint_as_float(w[q][j] << 16);
            b -= __uint_as_float(w[q][j] & 0xffff0000u);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (EDGE == 2) w[0][j] = dyr[v][2 * j] | dyr[v][2 * j + 1] << 16;
          else w[0][j] = dyr[v][j];
        }
      }
#pragma unroll
      for (int q = 0; q < P; ++q) *(uint4 *)(sd + (buf * P + q) * DBYTES + at) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
    }
  };

  a8_f32x16 acc[KG][NB];
#pragma unroll
  for (int u = 0; u < KG; ++u)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[u][n][r] = 0.f;

#pragma unroll
  for (int u = 0; u < KG; ++u) load_idx(u);
  load_dy();
  __builtin_amdgcn_sched_barrier(0);  // (in this order, as in the loop: the waits at its top count the loads behind dy's)
#pragma unroll
  for (int u = 0; u < KG; ++u) {
    load_code(u, 0);
    load_idx(u);
  }
  // the codes of unit u of chunk `of` into the half `h` of A; then its next loads (the index arrived a chunk ago)
  auto stage = [&](int u, int of, int h) {
    *(uint4 *)(sa + (h * UB + u % UB) * ABYTES + wg8_slot<64>(srow, sseg)) = wg8_restore<FMT>(code[u], sc[u]);
    load_code(u, of + 1);
    load_idx(u);
  };
  constexpr int PH = KG / UB;
  write_dy(0);
  load_dy();
#pragma unroll
  for (int u = 0; u < UB; ++u) stage(u, 0, 0);
  d3d_lds_barrier();
  // A phase multiplies UB units and meanwhile stages the next UB (behind the chunk's last: the next chunk's first, and its dy).
  // Written with the vector work between the MFMAs, which leave its pipe free: done one after the other, MFMA, restoring and
  // LDS add up (43 + 47 + 27 thousand cycles at 64 -> 64 channels, f32, where a CU is now busy for 100).
  for (int chunk = 0; chunk < chunks; ++chunk) {
    a8_bf16x8 bf[KS][NB][P];
    const unsigned char *const dcur = sd + (chunk & 1) * P * DBYTES;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < P; ++q) bf[k][n][q] = wg8_fragment<TN>(dcur + q * DBYTES, (wk * KS + k) * 16, (wco * NB + n) * 32);
#pragma unroll
    for (int ph = 0; ph < PH; ++ph) {
      const int h = PH % 2 == 0 ? ph & 1 : chunk & 1;  // this phase's half of A
      a8_bf16x8 af[UB][KS];
#pragma unroll
      for (int v = 0; v < UB; ++v)
#pragma unroll
        for (int k = 0; k < KS; ++k) af[v][k] = wg8_fragment<64>(sa + (h * UB + v) * ABYTES, (wk * KS + k) * 16, wci * 32);
      // (units behind the last are worked on too, with zeros: a branch around them would make every wait for a load a wait for all)
      if (ph + 1 < PH) {
#pragma unroll
        for (int v = 0; v < UB; ++v) stage((ph + 1) * UB + v, chunk, h ^ 1);
      } else {
        write_dy((chunk + 1) & 1);
        load_dy();
#pragma unroll
        for (int v = 0; v < UB; ++v) stage(v, chunk + 1, h ^ 1);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int q = P - 1; q >= 0; --q)
#pragma unroll
          for (int v = 0; v < UB; ++v)
#pragma unroll
            for (int n = 0; n < NB; ++n)
              acc[ph * UB + v][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[v][k], bf[k][n][q], acc[ph * UB + v][n], 0, 0, 0);
      WG8_INTERLEAVE
      d3d_lds_barrier();
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // ---- the parts of the chunk's rows (wk) together, then out: lane l holds column l % 32 of dy's 32, rows 8 (r / 4) + 4 (l / 32) + r % 4
#pragma unroll
  for (int u = 0; u < KG; ++u) {
    if (u >= nu) continue;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if constexpr (WK > 1) {
        float *red = (float *)smem;
        if (wk > 0) {
#pragma unroll
          for (int r = 0; r < 16; ++r) red[(((wk - 1) * 2 * WCO + (wave & (2 * WCO - 1))) * 16 + r) * 64 + lane] = acc[u][n][r];
        }
        d3d_lds_barrier();
        if (wk == 0) {
#pragma unroll
          for (int q = 0; q < WK - 1; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[u][n][r] += red[((q * 2 * WCO + wave) * 16 + r) * 64 + lane];
        }
        d3d_lds_barrier();
        if (wk > 0) continue;
      }
      const int co = co0 + (wco * NB + n) * 32 + (lane & 31);
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {  // four neighbouring columns of one offset
        const int col = (unit0 + u) * 64 + wci * 32 + r4 * 8 + ((lane >> 5) << 2);
        const int k = col / p.cinp, c = col - k * p.cinp;
        float *dst = p.out + split * p.count + ((int64_t)k * p.cin + c) * p.cout + co;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col < p.cols && c + r < p.cin && co < p.cout) dst[(int64_t)r * p.cout] = acc[u][n][r4 * 4 + r];
      }
    }
  }
}

// the row ranges' sums in their order: PARTS parts of the ranges side by side, then the parts.  Bound by latency where there are
// many ranges and few weights ([27, 16, 16], 128 ranges: 9.8 us with 4 parts, 3.9 with 16; [27, 64, 64], 36 ranges: 4.8 and 7.1),
// by HBM where there are few and many (4 MB of weights, 16 ranges: 10.6 us; 15.9 with one load of a thread in flight)
template <int PARTS>
__global__ void __launch_bounds__(64 * PARTS) a8_fold_kernel(const float *__restrict__ part, int64_t count, int splits, float *__restrict__ out) {
  __shared__ float sum[PARTS][64];
  const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int q = threadIdx.x >> 6, per = (splits + PARTS - 1) / PARTS;
  float s = 0.f;
  if (i < count) {
    const int last = (q + 1) * per < splits ? (q + 1) * per : splits;
#pragma unroll 4
    for (int k = q * per; k < last; ++k) s += part[k * count + i];
  }
  sum[q][threadIdx.x & 63] = s;
  __syncthreads();
  if (q != 0 || i >= count) return;
  float t[PARTS];
#pragma unroll
  for (int k = 0; k < PARTS; ++k) t[k] = sum[k][threadIdx.x];
#pragma unroll
  for (int m = 1; m < PARTS; m <<= 1)
#pragma unroll
    for (int k = 0; k < PARTS; k += 2 * m) t[k] += t[k + m];
  out[i] = t[0];
}

// How a weight gradient is cut: columns of dy a block, units, row ranges.  One block to a CU (256): at 64 -> 64 channels two took
// 58 to 61 us, half of them 62 (with 57 for one); two units to a block where there are no more than two to fill it
// (bf16 rows whose width is no multiple of 8 keep to 128 columns: shifting needs registers that the tile of 256 has not.
// [16000, 511] x [16000, 509]: 38 us, with 256 columns 51; f32 51 us.  Loaded value by value: 48, f32 69)
struct Wg8Plan {
  int tn, kg, edge, units, groups, cotiles, chunks, per_split, splits;
};
#define WG8_UB 2
static Wg8Plan wg8_plan(int64_t n_out, int kvol, int cin, int cout, int dtype, bool table) {
  Wg8Plan q;
  q.edge = cout % 8 == 0 ? 0 : (cout >= 8 ? 1 : 2);
  q.tn = cout <= 32 ? 32 : (cout <= 64 ? 64 : (cout <= 128 || dtype == D3D_F32 || q.edge ? 128 : 256));
  q.units = (int)(((int64_t)kvol * ((cin + 7) / 8 * 8) + 63) / 64);
  q.kg = q.units <= 2 && !table ? 2 : 4;
  q.groups = (q.units + q.kg - 1) / q.kg;
  q.cotiles = (cout + q.tn - 1) / q.tn;
  q.chunks = (int)((n_out + WG8_ROWS - 1) / WG8_ROWS);
  const int64_t tiles = (int64_t)q.groups * q.cotiles;
  int64_t s = 256 / tiles;
  s = s < 1 ? 1 : (s > q.chunks ? q.chunks : s);
  q.per_split = (int)((q.chunks + s - 1) / s);
  q.splits = (q.chunks + q.per_split - 1) / q.per_split;
  return q;
}

extern "C" size_t d3d_act8_wgrad_workspace_bytes(int64_t n_out, int kvol, int cin, int cout, int dtype) {
  if (n_out < 1 || kvol < 1 || cin < 1 || cout < 1 || (dtype != D3D_F32 && dtype != D3D_BF16)) return 0;
  // (with and without a table: the larger of the two)
  const int s0 = wg8_plan(n_out, kvol, cin, cout, dtype, true).splits, s1 = wg8_plan(n_out, kvol, cin, cout, dtype, false).splits;
  const int splits = s0 > s1 ? s0 : s1;
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
  D3D_REQUIRE((int64_t)kvol * cin * cout < ((int64_t)1 << 30), "d3d_act8_wgrad: a weight of %d x %d x %d", kvol, cin, cout);
  D3D_REQUIRE(n_in < ((int64_t)1 << 31) - 4096 && n_out < ((int64_t)1 << 31) - 4096, "d3d_act8_wgrad: %lld / %lld rows", (long long)n_in, (long long)n_out);
  D3D_REQUIRE(codes && scales && dy && dw, "d3d_act8_wgrad: null pointer");
  D3D_REQUIRE(dy_stride >= cout, "d3d_act8_wgrad: rows of %d channels %lld elements apart", cout, (long long)dy_stride);
  D3D_REQUIRE(nbr ? cap >= n_out : (kvol == 1 && n_in == n_out), "d3d_act8_wgrad: cap=%lld kvol=%d n_in=%lld n_out=%lld",
              (long long)cap, kvol, (long long)n_in, (long long)n_out);
  D3D_REQUIRE(!nbr || (n_in * a8_pitch(cin) < ((int64_t)1 << 31) - 16 && n_in < (1 << 24) && kvol * cap < (1 << 29)),
              "d3d_act8_wgrad: %lld held rows of %d channels behind a table of %d x %lld entries (below 2^24 rows, 2 GB of codes, 2 GB of table)",
              (long long)n_in, cin, kvol, (long long)cap);
  const size_t need = d3d_act8_wgrad_workspace_bytes(n_out, kvol, cin, cout, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return d3d_set_error(D3D_ECAPACITY, "d3d_act8_wgrad: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const Wg8Plan q = wg8_plan(n_out, kvol, cin, cout, dtype, nbr != nullptr);
  Wg8Args p;
  p.codes = codes;
  p.scales = scales;
  p.dy = dy;
  p.nbr = nbr;
  p.out = q.splits > 1 ? (float *)workspace : dw;
  p.dy_stride = dy_stride;
  p.cap = cap;
  p.count = (int64_t)kvol * cin * cout;
  p.n_in = (uint32_t)n_in;
  p.tab_bytes = nbr ? (uint32_t)(kvol * cap * 4) : 0u;
  p.n_out = (int)n_out;
  p.cin = cin;
  p.cinp = (cin + 7) / 8 * 8;
  p.pitch = a8_pitch(cin);
  p.cout = cout;
  p.cols = kvol * p.cinp;
  p.units = q.units;
  p.groups = q.groups;
  p.cotiles = q.cotiles;
  p.chunks = q.chunks;
  p.per_split = q.per_split;
  const dim3 grid((unsigned)(q.groups * q.cotiles * q.splits));
#define A8_WG(F, P, WCO, WK, NB, EDGE)                                                                                                    \
  do {                                                                                                                                    \
    if (nbr) hipLaunchKernelGGL((a8_wgrad_kernel<F, P, WCO, WK, NB, 4, WG8_UB, true, EDGE>), grid, dim3(512), 0, stream, p);              \
    else if (q.kg == 2) hipLaunchKernelGGL((a8_wgrad_kernel<F, P, WCO, WK, NB, 2, WG8_UB, false, EDGE>), grid, dim3(512), 0, stream, p);  \
    else hipLaunchKernelGGL((a8_wgrad_kernel<F, P, WCO, WK, NB, 4, WG8_UB, false, EDGE>), grid, dim3(512), 0, stream, p);                 \
  } while (0)
#define A8_WG_TN(F, P, EDGE)                                                                                                              \
  do {                                                                                                                                    \
    if (q.edge == 2) A8_WG(F, P, 1, 4, 1, 2);                                                                                             \
    else if (q.tn == 32) A8_WG(F, P, 1, 4, 1, EDGE);                                                                                      \
    else if (q.tn == 64) A8_WG(F, P, 2, 2, 1, EDGE);                                                                                      \
    else if (q.tn == 128) A8_WG(F, P, 4, 1, 1, EDGE);                                                                                     \
    else if constexpr (P == 1 && !EDGE) A8_WG(F, P, 4, 1, 2, EDGE);                                                                      \
  } while (0)
#define A8_WG_ALL(F)                                                                                                                      \
  do {                                                                                                                                    \
    if (dtype == D3D_BF16 && !q.edge) A8_WG_TN(F, 1, 0);                                                                                  \
    else if (dtype == D3D_BF16) A8_WG_TN(F, 1, 1);                                                                                        \
    else if (!q.edge) A8_WG_TN(F, 3, 0);                                                                                                  \
    else A8_WG_TN(F, 3, 1);                                                                                                               \
  } while (0)
  if (fmt == D3D_ACT8_INT8) A8_WG_ALL(D3D_ACT8_INT8);
  else A8_WG_ALL(D3D_ACT8_E4M3);
#undef A8_WG_ALL
#undef A8_WG_TN
#undef A8_WG
  D3D_LAUNCH_TRY("a8_wgrad_kernel");
  if (q.splits > 1) {
    const dim3 columns((unsigned)((p.count + 63) / 64));
    if (q.splits > 32 && columns.x <= 256) hipLaunchKernelGGL(a8_fold_kernel<16>, columns, dim3(1024), 0, stream, (const float *)workspace, p.count, q.splits, dw);
    else hipLaunchKernelGGL(a8_fold_kernel<4>, columns, dim3(256), 0, stream, (const float *)workspace, p.count, q.splits, dw);
    D3D_LAUNCH_TRY("a8_fold_kernel");
  }
  return D3D_OK;
}
