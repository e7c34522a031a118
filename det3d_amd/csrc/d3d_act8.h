// Rows held in 8 bits (include/d3d.h, d3d_act8_*): the arithmetic that the hold / restore kernels, the row norms and the weight
// gradient share, and the row vectors they move.
//
// 32 consecutive channels of a row form a group with one scale 2^s, stored as the biased exponent s + 127.  Powers of two make
// x 2^-s and code 2^s exact, so which code a value gets depends on the value alone (no rounding in front of the rounding), and a
// restored value has at most 8 significant bits: exact in bf16.
#pragma once
#include "d3d_common.h"

#define A8_GROUP 32

static inline int a8_pitch(int c) { return (c + A8_GROUP - 1) / A8_GROUP * A8_GROUP; }

// biased exponent of a group's scale from the bits of its largest |x| (0xff: the group holds a NaN or an infinity).
//   int8: rint(top 2^-s) <= 127  <=>  top 2^-s < 127.5 = 2^6 * 1.9921875 (the tie goes to the even 128): exponent - 6, one more
//         from mantissa 0x7f0000 on;   e4m3: top 2^-s <= 448 = 2^8 * 1.75: exponent - 8, one more above mantissa 0x600000
// The limits keep 2^-s and every code times 2^s normal and finite.
template <int FMT> __device__ __forceinline__ uint32_t a8_scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return 0xffu;
  int b = FMT == D3D_ACT8_INT8 ? (int)((top + 0x010000u) >> 23) - 6 : (int)((top + 0x1fffffu) >> 23) - 8;
  constexpr int LO = FMT == D3D_ACT8_INT8 ? 127 - 120 : 127 - 110, HI = FMT == D3D_ACT8_INT8 ? 127 + 121 : 127 + 119;
  return (uint32_t)(b < LO ? LO : (b > HI ? HI : b));
}
// 2^-s; 0 for a group of NaN (its codes are then zero, see a8_code4)
__device__ __forceinline__ float a8_down(uint32_t b) { return b == 0xffu ? 0.f : __uint_as_float((254u - b) << 23); }
// 2^s; infinity for 0xff, so that a zero code is restored as NaN
__device__ __forceinline__ float a8_up(uint32_t b) { return __uint_as_float(b << 23); }

// four codes in one word, value j in byte j
template <int FMT> __device__ __forceinline__ uint32_t a8_code4(const float *v, float down) {
  if (down == 0.f) return 0u;
  if constexpr (FMT == D3D_ACT8_INT8) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float q = fminf(fmaxf(rintf(v[j] * down), -127.f), 127.f);
      w |= ((uint32_t)(int)q & 0xffu) << (8 * j);
    }
    return w;
  } else {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = fminf(fmaxf(v[j] * down, -448.f), 448.f);  // (the clip acts at the upper limit of s only)
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  }
}
template <int FMT> __device__ __forceinline__ void a8_value4(uint32_t w, float up, float *v) {
  if constexpr (FMT == D3D_ACT8_INT8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)((int)(w << (24 - 8 * j)) >> 24) * up;
  } else {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0] * up;
    v[1] = a[1] * up;
    v[2] = b[0] * up;
    v[3] = b[1] * up;
  }
}

// 4, 8 or 16 bytes at any address: one load / store on gfx950 (unaligned access mode), the same as an aligned one
template <class V> __device__ __forceinline__ V a8_get(const void *p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <class V> __device__ __forceinline__ void a8_put(void *p, const V &v) { __builtin_memcpy(p, &v, sizeof(V)); }

typedef __attribute__((ext_vector_type(2))) float a8_f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 a8_bf16x2;
__device__ __forceinline__ uint32_t a8_pack_bf16(float a, float b) {  // round to nearest even
  const a8_f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, a8_bf16x2));
}

// E neighbouring values of a row in the feature type: one 16-byte access (E = 4 f32 / 8 bf16), or one value (E = 1).  Raw is
// what a load leaves in registers: loads issued early and unpacked late stay in flight in between.
template <bool BF16, int E> struct A8Row {
  static_assert(E == 1 || E == (BF16 ? 8 : 4), "one value or one 16-byte vector");
  struct Raw {
    uint32_t w[E == 1 ? 1 : 4];
  };
  __device__ static __forceinline__ Raw fetch(const void *row, int64_t at) {
    Raw r;
    if constexpr (E == 1) {
      if constexpr (BF16) r.w[0] = (uint32_t)((const uint16_t *)row)[at] << 16;
      else r.w[0] = ((const uint32_t *)row)[at];
    } else {
      const uint4 q = *(const uint4 *)((const char *)row + at * (BF16 ? 2 : 4));
      r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
    }
    return r;
  }
  __device__ static __forceinline__ Raw zero() {
    Raw r;
#pragma unroll
    for (uint32_t &w : r.w) w = 0u;
    return r;
  }
  __device__ static __forceinline__ void unpack(const Raw &r, float *v) {
    if constexpr (E > 1 && BF16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(r.w[j] << 16);
        v[2 * j + 1] = __uint_as_float(r.w[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = __uint_as_float(r.w[j]);
    }
  }
  __device__ static __forceinline__ void load(const void *row, int64_t at, float *v) { unpack(fetch(row, at), v); }
  // The same on rows of any alignment and any width c, for vectors that begin inside the row: one that passes its end is read as
  // the row's last E values and shifted into place (zeros behind the end), and written value by value.  hold of [100000, 127]:
  // f32 26 us, bf16 20 us (one value a lane and load: 55 and 55; rows of 128: 24 and 17)
  __device__ static __forceinline__ Raw fetch_any(const void *row, int at, int c) {
    constexpr int EB = BF16 ? 2 : 4;
    Raw r = zero();
    if (c >= E) {
      const uint4 q = a8_get<uint4>((const char *)row + (at + E <= c ? at : c - E) * EB);
      r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
    } else {  // (a row shorter than a vector)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (at + j >= c) continue;
        if constexpr (BF16) r.w[j / 2] |= (uint32_t)((const uint16_t *)row)[at + j] << (j % 2 * 16);
        else r.w[j] = ((const uint32_t *)row)[at + j];
      }
    }
    return r;
  }
  __device__ static __forceinline__ void unpack_any(const Raw &r, int at, int c, float *v) {
    unpack(r, v);
    const int s = at + E - c;
    if (s > 0 && c >= E) {
#pragma unroll
      for (int m = 1; m < E; m <<= 1)
        if (s & m) {
#pragma unroll
          for (int j = 0; j < E; ++j) v[j] = j + m < E ? v[j + m] : 0.f;
        }
    }
  }
  __device__ static __forceinline__ void store_any(void *row, int at, int c, const float *v) {
    constexpr int EB = BF16 ? 2 : 4;
    if (at + E <= c) {
      uint4 q;
      if constexpr (BF16) q = make_uint4(a8_pack_bf16(v[0], v[1]), a8_pack_bf16(v[2], v[3]), a8_pack_bf16(v[4], v[5]), a8_pack_bf16(v[6], v[7]));
      else q = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      a8_put((char *)row + at * EB, q);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (at + j < c) {
          if constexpr (BF16) ((uint16_t *)row)[at + j] = (uint16_t)(a8_pack_bf16(v[j], 0.f) & 0xffffu);
          else ((float *)row)[at + j] = v[j];
        }
    }
  }
  // one of the two: ANY = rows of any alignment and width
  template <bool ANY> __device__ static __forceinline__ Raw get(const void *row, int at, int c) {
    if constexpr (ANY) return fetch_any(row, at, c);
    else return fetch(row, at);
  }
  template <bool ANY> __device__ static __forceinline__ void open(const Raw &r, int at, int c, float *v) {
    if constexpr (ANY) unpack_any(r, at, c, v);
    else unpack(r, v);
  }
  template <bool ANY> __device__ static __forceinline__ void put(void *row, int at, int c, const float *v) {
    if constexpr (ANY) store_any(row, at, c, v);
    else store(row, at, v);
  }
  __device__ static __forceinline__ void store(void *row, int64_t at, const float *v) {
    if constexpr (E == 1) {
      if constexpr (BF16) ((uint16_t *)row)[at] = (uint16_t)(a8_pack_bf16(v[0], 0.f) & 0xffffu);
      else ((float *)row)[at] = v[0];
    } else if constexpr (BF16) {
      *(uint4 *)((uint16_t *)row + at) =
          make_uint4(a8_pack_bf16(v[0], v[1]), a8_pack_bf16(v[2], v[3]), a8_pack_bf16(v[4], v[5]), a8_pack_bf16(v[6], v[7]));
    } else {
      *(float4 *)((float *)row + at) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
};

// v combined over the T neighbouring lanes of a group, the same bits in every one of them (op commutes).  Steps of 1, 2, 4, 8 are
// operand modifiers of the operation itself (lanes that agree already stand in for one another, so a mirrored row is a step),
// 16 and 32 one instruction beside it: a dozen cycles a step, where a shuffle goes through LDS.
template <int CTRL> __device__ __forceinline__ uint32_t a8_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int T, class Op> __device__ __forceinline__ uint32_t a8_lanes(uint32_t v, Op op) {
  if constexpr (T > 1) v = op(v, a8_dpp<0xb1>(v));   // 1 0 3 2
  if constexpr (T > 2) v = op(v, a8_dpp<0x4e>(v));   // 2 3 0 1
  if constexpr (T > 4) v = op(v, a8_dpp<0x141>(v));  // 8 lanes mirrored
  if constexpr (T > 8) v = op(v, a8_dpp<0x140>(v));  // 16 lanes mirrored
  if constexpr (T > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if constexpr (T > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  return v;
}

// E values of a held row: LANES neighbouring lanes, each with E values, share a group (LANES * E = 32, or fewer where the
// whole row is shorter)
template <int FMT, int E, int LANES> struct A8Held {
  // codes[at .. at + E) and, by the group's first lane, its scale; every lane of the group takes part
  __device__ static __forceinline__ void store(uint8_t *codes, uint8_t *scales, int64_t row, int pitch, int at, bool inside,
                                               const float *v) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const uint32_t u = __float_as_uint(v[j]) & 0x7fffffffu;
      top = u > top ? u : top;
    }
    top = a8_lanes<LANES>(top, [](uint32_t l, uint32_t r) { return l > r ? l : r; });
    const uint32_t b = a8_scale_of<FMT>(top);
    const float down = a8_down(b);
    if (!inside) return;
    uint8_t *c = codes + row * pitch + at;
    if constexpr (E == 4) {
      *(uint32_t *)c = a8_code4<FMT>(v, down);
    } else {
      *(uint2 *)c = make_uint2(a8_code4<FMT>(v, down), a8_code4<FMT>(v + 4, down));
    }
    if ((at & (A8_GROUP - 1)) == 0) scales[row * (pitch / A8_GROUP) + at / A8_GROUP] = (uint8_t)b;
  }
  struct Raw {
    uint32_t w[E == 8 ? 2 : 1], b;
  };
  __device__ static __forceinline__ Raw fetch(const uint8_t *codes, const uint8_t *scales, int64_t row, int pitch, int at) {
    Raw r;
    r.b = scales[row * (pitch / A8_GROUP) + at / A8_GROUP];
    const uint8_t *c = codes + row * pitch + at;
    if constexpr (E == 4) r.w[0] = *(const uint32_t *)c;
    else {
      const uint2 q = *(const uint2 *)c;
      r.w[0] = q.x;
      r.w[1] = q.y;
    }
    return r;
  }
  __device__ static __forceinline__ Raw zero() {
    Raw r;
#pragma unroll
    for (uint32_t &w : r.w) w = 0u;
    r.b = 0u;
    return r;
  }
  __device__ static __forceinline__ void unpack(const Raw &r, float *v) {
    const float up = a8_up(r.b);
#pragma unroll
    for (int j = 0; j < E / 4; ++j) a8_value4<FMT>(r.w[j], up, v + 4 * j);
  }
  __device__ static __forceinline__ void load(const uint8_t *codes, const uint8_t *scales, int64_t row, int pitch, int at,
                                              float *v) {
    unpack(fetch(codes, scales, row, pitch, at), v);
  }
};

// may rows of `elem_bytes` elements at p, `stride` elements apart and c wide, be moved as 16-byte vectors?
static inline bool a8_vectors(const void *p, int64_t stride, int c, int elem_bytes) {
  const int e = 16 / elem_bytes;
  return p == nullptr || (((uintptr_t)p & 15) == 0 && stride % e == 0 && c % e == 0);
}
