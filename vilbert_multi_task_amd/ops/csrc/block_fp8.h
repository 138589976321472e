// 8-bit (OCP e4m3) values with one scale per block of 128, in bf16 or f32: what the
// norms, the quantisers and the products that share this format have in common.
//
//   a = max |v| over the block's finite v    s = held(max(a / 448, 2^-100))
//   q = e4m3(v * (1 / s)), to nearest even   v ~ q * s
//
// A scale in bf16 is half the bytes, and q is computed with the scale as it is
// held, so that its rounding is hardly an error of the value: only where it went
// down, a block's largest |q| comes to 449.75 at most and is stored as 448, 0.4%
// less. In f32 the scale is a / 448 itself and the largest |q| is 448.
// A value that is not finite is stored as e4m3's NaN and leaves its block's
// scale alone, so it reaches the results that it belongs to and no others.
// 2^-100 keeps 1/s finite where a block is all zeros.
#pragma once

#include "common.h"

constexpr int kBlock = 128;  // values under one scale

// rows of 8-bit values begin at multiples of 16 bytes
__host__ __device__ static inline long fp8_pitch(long k) { return (k + 15) / 16 * 16; }


// max |v| of N values, those that are not finite left out: fmaxf passes NaN
// over, and infinity is looked for only where it came out on top.
template <int N>
DEV float absmax(const float* v) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) a = fmaxf(a, fabsf(v[i]));
  if (a == INFINITY) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float b = fabsf(v[i]);
      a = fmaxf(a, b < INFINITY ? b : 0.f);
    }
  }
  return a;
}

// 4 values -> 4 e4m3 bytes. |v * inv| < 464 for finite v, which the conversion
// rounds to 448 at most; infinity and NaN it takes to NaN.
DEV unsigned int pack4_e4m3(float a, float b, float c, float d, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
  return (unsigned int)r;
}
DEV uint2 pack8_block(const float* v, float inv) {
  return make_uint2(pack4_e4m3(v[0], v[1], v[2], v[3], inv),
                    pack4_e4m3(v[4], v[5], v[6], v[7], inv));
}

// 8 neighbours of a row, wherever it begins: the type's own alignment is all
// that is promised, which the hardware's wide accesses take as they are.
struct __attribute__((packed, aligned(2))) U16x8 { unsigned int w[4]; };
struct __attribute__((packed, aligned(4))) F32x8 { float f[8]; };

// two f32 -> two bf16, to nearest even, NaN kept (one instruction on gfx950)
DEV unsigned int pack2_bf16(float a, float b) {
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  using b16x2 = __attribute__((ext_vector_type(2))) __bf16;
  const b16x2 r = __builtin_convertvector((f32x2){a, b}, b16x2);
  return __builtin_bit_cast(unsigned int, r);
}

// the scale of a block, as it is held in f32 or in bf16, from its largest value
template <bool F32>
DEV float block_scale(float amax) {
  const float s = fmaxf(amax / 448.0f, 0x1p-100f);
  return F32 ? s : us2f((unsigned short)pack2_bf16(s, s));
}
// number i of `scales`, of block_scale: nothing to round
template <bool F32>
DEV void store_scale(void* scales, long i, float scale) {
  if (F32)
    ((float*)scales)[i] = scale;
  else
    ((unsigned short*)scales)[i] = (unsigned short)(__float_as_uint(scale) >> 16);
}

DEV void load8u(const bf16* p, float* out) {
  const U16x8 raw = *reinterpret_cast<const U16x8*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[2 * i] = us2f((unsigned short)(raw.w[i] & 0xffff));
    out[2 * i + 1] = us2f((unsigned short)(raw.w[i] >> 16));
  }
}
DEV void load8u(const float* p, float* out) {
  const F32x8 raw = *reinterpret_cast<const F32x8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = raw.f[i];
}
DEV void store8u(bf16* p, const float* in) {
  U16x8 raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) raw.w[i] = pack2_bf16(in[2 * i], in[2 * i + 1]);
  *reinterpret_cast<U16x8*>(p) = raw;
}
DEV void store8u(float* p, const float* in) {
  F32x8 raw;
#pragma unroll
  for (int i = 0; i < 8; ++i) raw.f[i] = in[i];
  *reinterpret_cast<F32x8*>(p) = raw;
}
DEV float ld1(const bf16* p) { return bf2f(*p); }
DEV float ld1(const float* p) { return *p; }
DEV void st1(bf16* p, float v) {
  *reinterpret_cast<unsigned short*>(p) = (unsigned short)pack2_bf16(v, v);
}
DEV void st1(float* p, float v) { *p = v; }

// columns [j, j+8) of a row of `dim`; what is past its end reads as zero and
// is not written
template <typename T>
DEV void load8_row(const T* row, int j, int dim, float* out) {
  if (j + 8 <= dim) {
    load8u(row + j, out);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = j + i < dim ? ld1(row + j + i) : 0.f;
  }
}
template <typename T>
DEV void store8_row(T* row, int j, int dim, const float* in) {
  if (j + 8 <= dim) {
    store8u(row + j, in);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < dim) st1(row + j + i, in[i]);
  }
}
// what T holds of v
DEV float held(float v, const bf16*) { return us2f((unsigned short)pack2_bf16(v, v)); }
DEV float held(float v, const float*) { return v; }
