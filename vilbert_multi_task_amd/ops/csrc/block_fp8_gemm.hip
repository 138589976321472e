// Products of block-scaled 8-bit rows:
//
//   y[m,n] = sum_b xs[m,b] * ws[n/128,b] * (sum_{k in block b} x8[m,k] * w8[n,k])
//            + bias[n],   optionally GELU(y) = y/2 * (1 + erf(y / sqrt 2))
//
// One matrix instruction, 16x16x128 in e4m3, covers a whole block of 128 of the
// shared axis, so the inner sum is an instruction's result and the scales are
// applied to it in 32 bits: 4 multiply-adds a lane for each instruction, half
// of the cycles that the instruction itself takes, on the other pipe.
//
// What the instruction rounds: it aligns 8 neighbouring products to the largest
// of them and drops what is below 2^-13 of it (measured; all e4m3 instructions
// of this card do), the sums of eights are f32. On normal values that is 1.5e-5
// of the result's 2-norm, with a few channels ten times as large 3e-5: a hundredth
// of bf16's step, and less of an 8-bit one. Where something leaves in 32 bits, y
// itself or the scales of an 8-bit y, the products are exact instead: e4m3 values
// are bf16 values, and of those four 16x16x32 instructions take the block, twice as
// long (measured: 1e-8 of the 2-norm for a block, 4e-8 for eight).
//
// W is the instruction's first operand and X its second: a lane's four results
// are then four neighbouring outputs of ONE row of X, which is what a store, a
// bias and a row's scale want. Both operands give a lane 32 neighbouring bytes
// of a row; the order of the 128 products within the sum is the same for both,
// whatever it is.

#include <type_traits>

#include "block_fp8.h"

namespace {

using i32x8 = __attribute__((ext_vector_type(8))) int;

enum Out { kBf16, kFp8, kF32 };

struct GemmArgs {
  const unsigned char *x, *w;  // rows at 16 bytes
  const void *xs, *ws;         // of the kernel's type of scales
  const void* bias;  // or null; bf16, or f32 where bias_f32
  void* y;
  void* ys;  // 8-bit output: its scales, of the type of the others
  long x_pitch, w_pitch;
  int m, n, k;
  bool gelu, bias_f32;
};

DEV float bias_at(const GemmArgs& a, int n) {
  if (!a.bias || n >= a.n) return 0.f;
  return a.bias_f32 ? ((const float*)a.bias)[n] : bf2f(((const bf16*)a.bias)[n]);
}

// The plain result of an instruction: scale operands of zero select its form
// without scales.
DEV f32x4 mfma128(i32x8 a, i32x8 b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// SF: scales are f32, else bf16. What is read of one, and its value:
template <bool SF>
using Held = std::conditional_t<SF, unsigned, unsigned short>;
template <bool SF>
DEV float scale_value(unsigned held) {
  return SF ? __uint_as_float(held) : us2f((unsigned short)held);
}
// The scale of a block's products. Where two scales' product passes f32's range it is
// f32's largest number, not infinity, which times a block sum of nothing would be NaN.
DEV float both_scales(float x, float w) {
  return __builtin_elementwise_minimum(x * w, 3.40282347e38f);
}

// What leaves in 32 bits has to be right in 32.
template <Out OUT, bool SF>
constexpr bool kExact = OUT == kF32 || (OUT == kFp8 && SF);

// A lane's 32 values of one operand's row as the instructions take them: e4m3, or
// bf16, into which e4m3 goes as it is, NaN included.
using bf16v2 = __attribute__((ext_vector_type(2))) __bf16;
using bf16v8 = __attribute__((ext_vector_type(8))) __bf16;
struct Bf16x32 { bf16v8 v[4]; };
template <bool EXACT>
using Operand = std::conditional_t<EXACT, Bf16x32, i32x8>;
template <bool EXACT>
DEV Operand<EXACT> operand(i32x8 raw) {
  if constexpr (EXACT) {
    Bf16x32 to;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bf16v2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], 1.f, false);
      const bf16v2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], 1.f, true);
      const int at = i % 2 * 4;
      to.v[i / 2][at] = a[0], to.v[i / 2][at + 1] = a[1];
      to.v[i / 2][at + 2] = b[0], to.v[i / 2][at + 3] = b[1];
    }
    return to;
  } else {
    return raw;
  }
}
DEV f32x4 block_product(const i32x8& a, const i32x8& b) { return mfma128(a, b); }
DEV f32x4 block_product(const Bf16x32& a, const Bf16x32& b) {
  f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], p, 0, 0, 0);
  return p;
}

// 16 bytes of a row from column k on, k a multiple of 16; zero past its end.
// Rows begin at multiples of 16 bytes, so a piece that holds one byte of the
// row is read whole (no page ends within it) and the rest of it masked.
DEV uint4 load16_row(const unsigned char* row, int k, int dim) {
  if (k >= dim) return make_uint4(0, 0, 0, 0);
  const uint4 v = *reinterpret_cast<const uint4*>(row + k);
  const int have = dim - k;
  if (have >= 16) return v;
  auto part = [have](unsigned int w, int at) {
    const int n = have - at;
    return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1);
  };
  return make_uint4(part(v.x, 0), part(v.y, 4), part(v.z, 8), part(v.w, 12));
}

DEV i32x8 load32_row(const unsigned char* row, int k, int dim) {
  const uint4 a = load16_row(row, k, dim), b = load16_row(row, k + 16, dim);
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w,
               (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// GELU(v) = max(v, 0) - |v| h with h = erfc(|v| / sqrt 2) / 2, of which log2 is
// all but a parabola: -log2 h is fitted by a polynomial of degree 7, so one
// exponential is all that it takes (11 instructions; the library's erf with its two
// ranges takes some 45). h is good to 4.3e-6 of itself up to |v| = 4, a five-hundredth
// of bf16's half step, to 3.6e-5 up to 6 and to 7.6e-4 up to 8. Beyond, where |v| h is
// below 1e-14, it is good for nothing but being small: two thirds too small at 12.
// |v| is bounded where |v| h is nothing, so that infinities come out as the limits. The minimum and the maximum are those that
// keep NaN, which also need no quieting of their operands.
// For what leaves in 32 bits the fit has degree 14 and goes to |v| = 12.9, beyond which
// h is no normal number of f32 and taken as 0: h is good to 1.3e-6 of itself up to 4,
// 1.4e-5 up to 8, 1.3e-3 at the end.
template <bool EXACT>
DEV float gelu(float v) {
  if constexpr (EXACT) {
    constexpr float c[] = {5.91124225e-14f, -5.77921784e-12f, 2.54662189e-10f,
                           -6.67860814e-9f, 1.15810212e-7f,   -1.3914505e-6f,
                           1.17169952e-5f,  -6.68080758e-5f,  2.13216115e-4f,
                           1.99831872e-4f,  -7.27495374e-3f,  5.27356344e-2f,
                           0.45909019f,     1.15112632f,      0.99999939f};
    const float a = __builtin_elementwise_minimum(fabsf(v), 14.f);
    float p = c[0];
#pragma unroll
    for (int i = 1; i < 15; ++i) p = p * a + c[i];
    return __builtin_elementwise_maximum(v, 0.f) - a * __builtin_amdgcn_exp2f(-p);
  }
  const float a = __builtin_elementwise_minimum(fabsf(v), 16.f);
  float p = 1.7221218e-6f;
  p = p * a - 5.9576460e-5f;
  p = p * a + 9.1649377e-4f;
  p = p * a - 8.4600993e-3f;
  p = p * a + 5.3876507e-2f;
  p = p * a + 0.45853566f;
  p = p * a + 1.1512260f;
  p = p * a + 0.99999761f;
  return __builtin_elementwise_maximum(v, 0.f) - a * __builtin_amdgcn_exp2f(-p);
}

struct __attribute__((packed, aligned(2))) B16x4 { unsigned int w[2]; };

DEV void store4(bf16* p, const float* v) {
  *reinterpret_cast<B16x4*>(p) = {{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3])}};
}
// Results go past the caches: kept there, a round of tiles' results would fill an
// XCD's whole cache and push out the W that the next round reads (103424x1024x1024
// by 256 x 128: 169 us with plain stores, 134 with these).
DEV void store16_past(void* p, uint4 v) {  // at any multiple of 2 bytes
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, (u32x4*)p);
}
// 8 neighbours of a row, as they are held
DEV void store8_row(bf16* row, int j, int dim, uint4 v) {
  if (j + 8 <= dim) {
    store16_past(row + j, v);
  } else {
    const unsigned int w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < dim)
        reinterpret_cast<unsigned short*>(row)[j + i] = w[i / 2] >> (16 * (i & 1));
  }
}
struct __attribute__((packed, aligned(4))) F32x4 { float f[4]; };
DEV void store4(float* p, const float* v) {
  *reinterpret_cast<F32x4*>(p) = {{v[0], v[1], v[2], v[3]}};
}
template <typename T>
DEV void store4_row(T* row, int j, int dim, const float* v) {
  if (j + 4 <= dim) {
    store4(row + j, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < dim) st1(row + j + i, v[i]);
  }
}

// --- few rows -----------------------------------------------------------------
//
// What counts is how long one read of memory takes, so every read is out at once:
// a workgroup has NT*16 outputs of MT*16 rows, and its 8 waves share the blocks of
// the shared axis out among them, straight from memory to the instruction, the
// next block's operands on their way while one is multiplied. Their sums are added
// through shared memory, in the order of the waves. (An 8-bit result needs 128
// outputs in one workgroup, and then reading them takes as long as with tiles.)
template <int NT, int MT, Out OUT, bool SF>
__global__ __launch_bounds__(512) void block_gemm_direct_kernel(GemmArgs a) {
  constexpr bool EXACT = kExact<OUT, SF>;
  constexpr int KW = 8;
  static_assert(NT * MT <= KW, "a wave for each part of the result");
  __shared__ f32x4 part[KW][NT * MT][64];
  const int lane = lane_id(), r = lane & 15, q = lane >> 4, kw = wave_id();
  const int ntiles = ceil_div(a.n, NT * 16);
  const int n0 = (blockIdx.x % ntiles) * NT * 16;
  const int m0 = (blockIdx.x / ntiles) * 16 * MT;
  const int kb = ceil_div(a.k, kBlock);

  // rows past the end are read as the last one and not written
  const unsigned char *wrow[NT], *xrow[MT];
  const Held<SF>* xs[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    wrow[t] = a.w + (long)min(n0 + t * 16 + r, a.n - 1) * a.w_pitch;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const long m = min(m0 + u * 16 + r, a.m - 1);
    xrow[u] = a.x + m * a.x_pitch;
    xs[u] = (const Held<SF>*)a.xs + m * kb;
  }
  const Held<SF>* const ws = (const Held<SF>*)a.ws + (long)(n0 / kBlock) * kb;

  i32x8 w[NT], x[MT];
  float s[MT];
  auto load = [&](int b) __attribute__((always_inline)) {
    const int k = b * kBlock + q * 32;
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = load32_row(wrow[t], k, a.k);
#pragma unroll
    for (int u = 0; u < MT; ++u) x[u] = load32_row(xrow[u], k, a.k);
    const float wsb = scale_value<SF>(ws[b]);
#pragma unroll
    for (int u = 0; u < MT; ++u) s[u] = both_scales(scale_value<SF>(xs[u][b]), wsb);
  };
  f32x4 acc[NT][MT] = {};
  if (kw < kb) load(kw);
  for (int b = kw; b < kb; b += KW) {
    Operand<EXACT> wb[NT], xb[MT];
    float sb[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wb[t] = operand<EXACT>(w[t]);
#pragma unroll
    for (int u = 0; u < MT; ++u) xb[u] = operand<EXACT>(x[u]), sb[u] = s[u];
    if (b + KW < kb) load(b + KW);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const f32x4 p = block_product(wb[t], xb[u]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][u][i] += p[i] * sb[u];
      }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) part[kw][t * MT + u][lane] = acc[t][u];
  __syncthreads();

  // wave kw has part kw of the outputs from here on
  const int n = n0 + (kw / MT) * 16 + q * 4, m = m0 + (kw % MT) * 16 + r;
  if (kw >= NT * MT || m >= a.m) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < KW; ++j) {
    const f32x4 p = part[j][kw][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += p[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] += bias_at(a, n + i);
    if (a.gelu) v[i] = gelu<EXACT>(v[i]);
  }
  using Y = std::conditional_t<OUT == kF32, float, bf16>;
  store4_row((Y*)a.y + (long)m * a.n, n, a.n, v);
}

// --- tiles through shared memory ---------------------------------------------
//
// A workgroup of WN x WM waves has WN*128 outputs of WM*MT*16 rows; a wave has
// 128 outputs (one block of W's scales, one block of an 8-bit result) of MT*16
// rows. For each block of the shared axis both operands' 128 bytes a row are
// copied straight from memory into shared memory; W has two buffers, X one: a
// wave takes its part of X into registers at once, and while it multiplies, the
// next block arrives. 256 outputs x 128 rows need 80 KB, so that two workgroups
// share a compute unit and one's loads, scaling and stores run beside the
// other's matrix instructions.
//
// Of a row's eight 16-byte pieces a lane multiplies number q and number q + 4, of
// both operands; the pieces are permuted within a row's 128 bytes by its number,
// so that lanes that read at once use all banks (with pieces 2q and 2q + 1, which
// the instruction's own order would suggest, reads take 1.4 times as long). X's
// rows go to the instruction in order; W's are dealt out so that a lane's results
// of two instructions are 8 neighbouring outputs and four lanes' 32.

// 16 bytes a lane from `base` + `offset` to shared memory at `lds` + 16 * lane.
// The compiler does not see that these write memory: stage_wait() comes before
// any reading of it.
// `lanes`: -1, all, or 0, none.
DEV void lds_load16(const unsigned char* base, unsigned offset, unsigned lds,
                    long lanes) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_mov_b64 exec, %3\n\t"
      "global_load_lds_dwordx4 %0, %1\n\t"
      "s_mov_b64 exec, -1"
      :: "v"(offset), "s"(base), "s"(lds), "s"(lanes)
      : "memory", "m0");
}
// this wave's loads have arrived and its reads are done; then everyone's
DEV void stage_wait() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
DEV void reads_done() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

DEV unsigned lds_address(const unsigned char* p) {
  return (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)p;
}

DEV int swizzle_w(int row) { return (row & 3) | ((row >> 1) & 4); }
DEV int swizzle_x(int row) { return row & 7; }

DEV i32x8 read_frag(const unsigned char* row, int q, int swz) {
  const uint4 a = *reinterpret_cast<const uint4*>(row + ((q ^ swz) << 4));
  const uint4 b = *reinterpret_cast<const uint4*>(row + (((q + 4) ^ swz) << 4));
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w,
               (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

template <typename T>
DEV T opaque(T v) {  // what the compiler is not to work out ahead and keep
  asm volatile("" : "+v"(v));
  return v;
}
// The last block of a width that is no multiple of 128, through registers, with
// zeros in place of what is past the end. `off` is
// where the thread's piece of a row is, `piece` what it is within the row.
template <int LOADS, int T>
DEV void stage_last(const unsigned char* base, const unsigned* off,
                    unsigned char* to, int k0, int piece, int k) {
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    *reinterpret_cast<uint4*>(to + (i * T + threadIdx.x % T) * 16) =
        load16_row(base + off[i] - piece, k0 + piece, k);
  }
}

// Where there are fewer tiles than compute units, KG = 2 such teams of waves share a
// tile: each has every other block of the shared axis, buffers of its own, and the
// second hands its sums to the first at the end.
template <int WN, int WM, int MT, int KG, Out OUT, bool SF>
__global__ __launch_bounds__(KG * WN * WM * 64,
                             MT == 4 || (MT == 2 && kExact<OUT, SF>) ? 2
                             : MT == 2                               ? 3
                                                                     : 4) void
block_gemm_tile_kernel(GemmArgs a, int mtiles, int ntiles) {
  constexpr bool EXACT = kExact<OUT, SF>;
  constexpr int T = WN * WM * 64;  // threads of a team
  constexpr int kN = WN * 128, kM = WM * MT * 16;
  constexpr int kStep = T / 8;  // rows that one load of all threads covers
  constexpr int kWLoads = kN / kStep, kXLoads = kM / kStep;
  // the fewer rows a wave has, the fewer instructions a step has to wait behind
  // (exact products take four times the instructions, and registers, a step)
  constexpr int kParts = EXACT || MT == 4 ? 2 : MT == 2 ? 3 : 4,
                kLag = EXACT || MT != 1 ? 1 : 2;
  // one load every so many matrix instructions
  constexpr int kEvery = 8 * MT / (kWLoads + kXLoads);
  static_assert(kEvery >= 1, "each load has its place");
  constexpr int kTeam = (2 * kN + kM) * 128;  // a team's shared memory
  extern __shared__ __attribute__((aligned(128))) unsigned char all[];

  // Workgroups go round the 8 XCDs, each with a cache of its own: each XCD gets
  // one stretch of tiles, W's tiles fastest (at most 16 of them before the next
  // of X's), so that it reads its part of X once and keeps W.
  int id = blockIdx.x;
  const int total = mtiles * ntiles;
  {
    const int per = total / 8, more = total % 8, xcd = id % 8;
    id = xcd * per + min(xcd, more) + id / 8;
  }
  const int strip = id / (16 * mtiles);
  const int width = min(16, ntiles - strip * 16);
  const int in = id - strip * 16 * mtiles;
  const int m0 = __builtin_amdgcn_readfirstlane((in / width) * kM);
  const int n0 = __builtin_amdgcn_readfirstlane((strip * 16 + in % width) * kN);

  const int tid = threadIdx.x % T, lane = lane_id(), r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(wave_id()) % (WN * WM);
  const int team = __builtin_amdgcn_readfirstlane(wave_id()) / (WN * WM);
  const int wn = wave % WN, wm = wave / WN;
  unsigned char* const smem = all + team * kTeam;
  unsigned char* const ldsx = smem + 2 * kN * 128;
  const int kb = ceil_div(a.k, kBlock);
  const int groups = ceil_div(a.n, kBlock);

  // what this thread copies: piece tid % 8 of rows tid / 8 + i * kStep. Rows
  // past the end are copied as the last one and not written.
  const unsigned char* const wbase = a.w + (long)n0 * a.w_pitch;
  const unsigned char* const xbase = a.x + (long)m0 * a.x_pitch;
  unsigned woff[kWLoads], xoff[kXLoads];
#pragma unroll
  for (int i = 0; i < kWLoads; ++i)
    woff[i] = min(tid / 8 + i * kStep, a.n - 1 - n0) * (unsigned)a.w_pitch +
              (((tid & 7) ^ swizzle_w(tid / 8)) << 4);
#pragma unroll
  for (int i = 0; i < kXLoads; ++i)
    xoff[i] = min(tid / 8 + i * kStep, a.m - 1 - m0) * (unsigned)a.x_pitch +
              (((tid & 7) ^ swizzle_x(tid / 8)) << 4);
  const unsigned lds0 =
      __builtin_amdgcn_readfirstlane(lds_address(all)) + team * kTeam + wave * 1024;

  const unsigned lds_x = lds0 + 2 * kN * 128;

  // Scales, of this lane's rows of X and of the wave's block of W, for four
  // blocks at a time: lanes of quarter q fetch the one of block b + q, and all get
  // it from there. Fetched block by block, 16 rows' lines each time for two bytes
  // of each, they cost as much of the first cache as half of X.
  const int group = min(n0 / kBlock + wn, groups - 1);
  const Held<SF>* const ws = (const Held<SF>*)a.ws + (long)group * kb;
  const Held<SF>* const xs = (const Held<SF>*)a.xs + (long)m0 * kb;
  unsigned xsoff[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    xsoff[t] = min((wm * MT + t) * 16 + r, a.m - 1 - m0) * kb;
  int xs4[MT], ws4;
  auto load_scales = [&](int b) __attribute__((always_inline)) {
    const int at = min(b + q * KG, kb - 1);
    ws4 = ws[at];
#pragma unroll
    for (int t = 0; t < MT; ++t) xs4[t] = xs[xsoff[t] + at];
  };

  f32x4 acc[8][MT] = {};
  float s[MT];
  Operand<EXACT> xf[MT];
  auto take_scales = [&](int b) __attribute__((always_inline)) {
    const int from = (b / KG & 3) * 16;
    const float w = scale_value<SF>(__builtin_amdgcn_readlane(ws4, from));
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      s[t] = both_scales(
          scale_value<SF>(__builtin_amdgcn_ds_bpermute((from + r) * 4, xs4[t])), w);
      // here and not later, where waiting for them would be waiting for W
      asm volatile("" : "+v"(s[t]));
    }
  };
  auto take_x = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
      xf[t] = operand<EXACT>(
          read_frag(ldsx + ((wm * MT + t) * 16 + r) * 128, q, swizzle_x(r)));
  };
  auto w_at = [](int b) { return (b / KG & 1) * kN * 128; };
  // The loads of a block, one at a time: W's first, then X's.
  auto load = [&](int b, int i, long lanes) __attribute__((always_inline)) {
    if (i < kWLoads)
      lds_load16(wbase + b * kBlock, woff[i], lds0 + w_at(b) + i * T * 16, lanes);
    else if (i < kWLoads + kXLoads)
      lds_load16(xbase + b * kBlock, xoff[i - kWLoads], lds_x + (i - kWLoads) * T * 16, lanes);
  };
  // W is read kParts steps ahead, and results are scaled kLag steps after their
  // instructions went out, while later ones run. The next
  // block's loads go out one by one between them: in a row they would fill the
  // queue and hold the wave, and with it its matrix instructions, up.
  auto multiply = [&](const unsigned char* wl, auto between)
      __attribute__((always_inline)) {
    auto part = [&](int t) __attribute__((always_inline)) {
      const int row = (t / 2) * 32 + (r / 4) * 8 + (t & 1) * 4 + (r & 3);
      return read_frag(wl + row * 128, q, swizzle_w((r / 4) * 8 + (r & 3)));
    };
    i32x8 wf[kParts];
    f32x4 p[kLag + 1][MT];
#pragma unroll
    for (int t = 0; t < kParts; ++t) wf[t] = part(t);
#pragma unroll
    for (int t = 0; t < kLag; ++t) {
      const Operand<EXACT> w = operand<EXACT>(wf[t]);
#pragma unroll
      for (int u = 0; u < MT; ++u) p[t][u] = block_product(w, xf[u]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if (t + kParts < 8) wf[t % kParts] = part(t + kParts);
      Operand<EXACT> w;
      if (t + kLag < 8) w = operand<EXACT>(wf[(t + kLag) % kParts]);
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        if (t + kLag < 8) p[(t + kLag) % (kLag + 1)][u] = block_product(w, xf[u]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][u][i] += p[t % (kLag + 1)][u][i] * s[u];
        if ((t * MT + u) % kEvery == 0) between((t * MT + u) / kEvery);
        __builtin_amdgcn_sched_barrier(0);  // in this order
      }
    }
  };

  const int whole = a.k / kBlock;
  // the last block of a width that is no multiple of 128
  auto load_last = [&](int b) __attribute__((always_inline)) {
    const int id = opaque(tid);
    stage_last<kWLoads, T>(wbase, woff, smem + w_at(b), b * kBlock,
                           ((id & 7) ^ swizzle_w(id / 8)) << 4, a.k);
    stage_last<kXLoads, T>(xbase, xoff, ldsx, b * kBlock,
                           ((id & 7) ^ swizzle_x(id / 8)) << 4, a.k);
  };
  // -1 where block b is to be copied, else 0; by hand, to be a scalar
  auto lanes_of = [&](int b) __attribute__((always_inline)) {
    int lanes;
    asm("s_sub_i32 %0, %1, %2\n\ts_ashr_i32 %0, %0, 31"
        : "=&s"(lanes) : "s"(b), "s"(whole) : "scc");
    return (long)lanes;
  };
  load_scales(team);
  if (team == whole && whole < kb) load_last(team);
#pragma unroll
  for (int i = 0; i < kWLoads + kXLoads; ++i) load(team, i, lanes_of(team));
  for (int block = 0; block < kb; block += KG) {
    const int b = __builtin_amdgcn_readfirstlane(block) + team;
    stage_wait();
    take_scales(b);
    take_x();
    reads_done();
    const int next = b + KG;
    const long lanes = lanes_of(next);
    if (next == whole && whole < kb) load_last(next);
    if ((b / KG & 3) == 3) load_scales(next);
    if (KG == 1 || b < kb)
      multiply(smem + w_at(b) + wn * 128 * 128,
               [&](int i) __attribute__((always_inline)) { load(next, i, lanes); });
  }
  reads_done();
  if (KG == 2) {
    f32x4* const sums = (f32x4*)(all + WN * WM * MT * 16 * 256) + wave * 8 * MT * 64 + lane;
    if (team == 1) {
#pragma unroll
      for (int i = 0; i < 8 * MT; ++i) sums[i * 64] = acc[i / MT][i % MT];
    }
    reads_done();
    if (team == 1) return;
#pragma unroll
    for (int i = 0; i < 8 * MT; ++i) acc[i / MT][i % MT] += sums[i * 64];
  }

  // acc[t][u][i]: output (t/2)*32 + q*8 + (t&1)*4 + i of row u*16 + r
  const int nw = n0 + wn * 128;
  if (a.bias) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float b8[8];
      if (a.bias_f32)
        load8_row((const float*)a.bias, nw + g * 32 + q * 8, a.n, b8);
      else
        load8_row((const bf16*)a.bias, nw + g * 32 + q * 8, a.n, b8);
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[2 * g + i / 4][u][i & 3] += b8[i];
    }
  }
  if (a.gelu) {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][u][i] = gelu<EXACT>(acc[t][u][i]);
  }
  if (nw >= a.n) return;
  if constexpr (OUT == kF32) {
    // Four lanes have a whole line of 128 bytes, and it goes past the caches (38912 x
    // 3072 x 768: 254 us with plain stores, 243 with these).
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const int m = m0 + (wm * MT + u) * 16 + r;
      if (m >= a.m) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = nw + g * 32 + q * 8;
        float* const row = (float*)a.y + (long)m * a.n;
        float v8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v8[i] = acc[2 * g + i / 4][u][i & 3];
        if (at + 8 <= a.n) {
          store16_past(row + at, __builtin_bit_cast(uint4, acc[2 * g][u]));
          store16_past(row + at + 4, __builtin_bit_cast(uint4, acc[2 * g + 1][u]));
        } else {
          ::store8_row(row, at, a.n, v8);
        }
      }
    }
    return;
  }
  // Out through shared memory, each wave through a part of its own, so that a
  // store instruction writes whole rows of 128 outputs. Pieces of 16 bytes change
  // places within a row by its number, as before.
  unsigned char* const out = all + wave * (MT * 16 * 256);
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int row = u * 16 + r;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = acc[i / 4][u][i & 3];
    if (OUT == kBf16) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint4*>(out + row * 256 + (((g * 4 + q) ^ r) << 4)) =
            make_uint4(pack2_bf16(v[8 * g], v[8 * g + 1]),
                       pack2_bf16(v[8 * g + 2], v[8 * g + 3]),
                       pack2_bf16(v[8 * g + 4], v[8 * g + 5]),
                       pack2_bf16(v[8 * g + 6], v[8 * g + 7]));
    } else {
      if (nw + kBlock > a.n) {  // what is past the end has no part in the scale
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (nw + (i / 8) * 32 + q * 8 + (i & 7) >= a.n) v[i] = 0.f;
      }
      float most = absmax<32>(v);
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      const float scale = block_scale<SF>(most), inv = 1.0f / scale;
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(out + row * 128 +
                                  (((g * 2 + q / 2) ^ (r & 7)) << 4) + (q & 1) * 8) =
            pack8_block(v + 8 * g, inv);
      const int m = m0 + wm * MT * 16 + row;
      if (q == 0 && m < a.m)
        store_scale<SF>(a.ys, (long)m * groups + nw / kBlock, scale);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int kRow = OUT == kBf16 ? 16 : 8;  // lanes that write a row
  const int piece = lane % kRow;
#pragma unroll
  for (int i = 0; i < MT * 16 * kRow / 64; ++i) {
    const int row = i * (64 / kRow) + lane / kRow;
    const int m = m0 + wm * MT * 16 + row;
    const uint4 v = *reinterpret_cast<const uint4*>(
        out + row * kRow * 16 + ((piece ^ (row & (kRow - 1))) << 4));
    if (m >= a.m) continue;
    if (OUT == kBf16) {
      store8_row((bf16*)a.y + (long)m * a.n, nw + piece * 8, a.n, v);
    } else if (nw + piece * 16 < a.n) {
      store16_past((unsigned char*)a.y + m * fp8_pitch(a.n) + nw + piece * 16, v);
    }
  }
}

template <int WN, int WM, int MT, int KG, Out OUT, bool SF>
void launch_tiles(const GemmArgs& a, hipStream_t stream) {
  constexpr int kLds = KG * (2 * WN * 128 * 128 + WM * MT * 16 * 128);
  static_assert(kLds >= WN * WM * MT * (16 * 256 + (KG - 1) * 8 * 1024),
                "room for the results");
  const int mtiles = ceil_div(a.m, WM * MT * 16), ntiles = ceil_div(a.n, WN * 128);
  hipLaunchKernelGGL((block_gemm_tile_kernel<WN, WM, MT, KG, OUT, SF>),
                     dim3(mtiles * ntiles), dim3(KG * WN * WM * 64), kLds, stream, a,
                     mtiles, ntiles);
}

// --- large products ----------------------------------------------------------
//
// One workgroup a compute unit, for as long as there are tiles: 8 waves on 256
// outputs x 256 rows, so that a third less is copied for each instruction than with
// 256 x 128, and the next tile's blocks arrive while a tile's results are written.
// A wave has 32 matrix instructions a block, and the two waves of a SIMD are to
// keep its matrix unit fed, so nothing may come in bursts that all wait for:
//   - there is one barrier a block, three quarters through it. By then every read
//     of this block's operands is done, the next block has arrived, and the last
//     eight instructions run under the reads of the next block's first operands;
//     this block's buffers take the block after next from there on.
//   - the instructions go by pairs of 16 outputs, rows within, so that W has eight
//     instructions' time to come from shared memory and X six.
//   - results are scaled two instructions after they went out.
//   - a copy is three scalar or vector instructions: all lanes are at work, m0 is
//     not kept, offsets are not worked out again (with twelve, 3700 cycles a block;
//     with three, 2900; the matrix unit needs 2048).
// Nothing that the compiler would wait for itself is loaded from memory on the way:
// the scales and the bias come through shared memory as well. What bounds it then is
// power: at 70% of the matrix unit's time the clock is down to 1.6 GHz of 2.4.
// 8192x8192x8192 447 us (2460 TFLOP/s; 256 x 128 515), 103424x1024x1024 126 (1720).
//
// Shared memory: two buffers of W and of X, two each of the rows' and W's scales
// and of the bias, and room for results on their way out.
constexpr int kWideW = 256 * 128, kWideScales = 2048, kWideBias = 1024;
constexpr int kWideOut = 4 * kWideW + 2 * kWideScales + 2 * kWideBias;
constexpr int kWideLds = kWideOut + 8 * 2048;
static_assert(kWideLds <= 160 * 1024, "one workgroup a compute unit");

// 16 bytes a lane from `base` + `offset` to shared memory at `lds` + TO + 16 * lane,
// and the same of one value of 2 or 4 bytes, to 4 * lane. All lanes are at work.
template <int TO>
DEV void wide_load16(const unsigned char* base, unsigned offset, unsigned lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(offset), "s"(base), "s"(lds), "n"(TO) : "memory", "m0", "scc");
}
DEV void wide_load2(const void* base, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ushort %0, %1"
               :: "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
DEV void wide_load4(const void* base, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :: "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}

// Widths that are multiples of 128 both ways, from 256 outputs, 256 rows and two
// blocks of the shared axis on.
template <Out OUT, bool SF>
__global__ __launch_bounds__(512, 2) void block_gemm_wide_kernel(GemmArgs a, int mtiles,
                                                                 int ntiles) {
  static_assert(!kExact<OUT, SF>, "its registers are full as it is");
  constexpr int kTurn = 24;  // the instruction before which the barrier is
  extern __shared__ __attribute__((aligned(128))) unsigned char all[];

  const int tid = threadIdx.x, lane = lane_id(), r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int wn = wave % 2, wm = wave / 2;
  const int kb = a.k / kBlock, groups = a.n / kBlock;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_address(all));
  const unsigned lds_w = lds0 + wave * 1024, lds_x = lds_w + 2 * kWideW;
  const unsigned lds_s = lds0 + 4 * kWideW + wave * 256;
  const unsigned lds_b = lds0 + 4 * kWideW + 2 * kWideScales + (wave & 3) * 256;

  // Each XCD has one stretch of the tiles, W's fastest, and its workgroups take
  // them in turn.
  const int total = mtiles * ntiles, xcd = blockIdx.x % 8;
  const int per = total / 8, more = total % 8;
  const int end = __builtin_amdgcn_readfirstlane((xcd + 1) * per + min(xcd + 1, more));
  const int step = __builtin_amdgcn_readfirstlane((gridDim.x - xcd + 7) / 8);
  const int first =
      __builtin_amdgcn_readfirstlane(xcd * per + min(xcd, more) + blockIdx.x / 8);

  // What is loaded next: block `lb` of tile `lt`, which is at m1, n1; at most one
  // tile ahead, and past the last tile the same again. A tile at the edge is moved
  // back by what it would stick out, so that a thread's offsets are the same for all
  // tiles; what its neighbour has is not written again.
  int lt = first, lb = 0, m1 = 0, n1 = 0;
  const unsigned char *wfrom = a.w, *xfrom = a.x;
  const Held<SF>* sfrom = nullptr;
  unsigned woff[4], xoff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    woff[i] = opaque((tid / 8 + i * 64) * (unsigned)a.w_pitch +
                     (((tid & 7) ^ swizzle_w(tid / 8)) << 4));
    xoff[i] = opaque((tid / 8 + i * 64) * (unsigned)a.x_pitch +
                     (((tid & 7) ^ swizzle_x(tid / 8)) << 4));
  }
  // waves 0 to 3 load the rows' scales, 4 W's, and the others do so for nothing
  const unsigned soff = opaque((wave < 4 ? tid : tid & 1) * kb * (int)sizeof(Held<SF>));
  auto enter = [&]() __attribute__((always_inline)) {
    const int strip = lt / (16 * mtiles);
    const int width = min(16, ntiles - strip * 16);
    const int in = lt - strip * 16 * mtiles;
    m1 = __builtin_amdgcn_readfirstlane((in / width) * 256);
    n1 = __builtin_amdgcn_readfirstlane((strip * 16 + in % width) * 256);
    const int m0 = min(m1, a.m - 256), n0 = min(n1, a.n - 256);
    wfrom = a.w + n0 * a.w_pitch;
    xfrom = a.x + m0 * a.x_pitch;
    sfrom = wave < 4 ? (const Held<SF>*)a.xs + (long)m0 * kb
                     : (const Held<SF>*)a.ws + (long)(n0 / kBlock) * kb;
  };
  auto next = [&]() __attribute__((always_inline)) {
    wfrom += kBlock;
    xfrom += kBlock;
    ++sfrom;
    if (++lb < kb) return;
    lb = 0;
    lt = min(lt + step, end - 1);
    enter();
  };
  auto load_x = [&](int i, int buf) __attribute__((always_inline)) {
    const unsigned to = lds_x + buf * kWideW;
    if (i == 0) wide_load16<0>(xfrom, xoff[0], to);
    if (i == 1) wide_load16<8192>(xfrom, xoff[1], to);
    if (i == 2) wide_load16<16384>(xfrom, xoff[2], to);
    if (i == 3) wide_load16<24576>(xfrom, xoff[3], to);
    if (i == 4 && SF) wide_load4(sfrom, soff, lds_s + buf * kWideScales);
    if (i == 4 && !SF) wide_load2(sfrom, soff, lds_s + buf * kWideScales);
  };
  auto load_w = [&](const unsigned char* from, int i, int buf)
      __attribute__((always_inline)) {
    const unsigned to = lds_w + buf * kWideW;
    if (i == 0) wide_load16<0>(from, woff[0], to);
    if (i == 1) wide_load16<8192>(from, woff[1], to);
    if (i == 2) wide_load16<16384>(from, woff[2], to);
    if (i == 3) wide_load16<24576>(from, woff[3], to);
  };
  // the bias of the tile at m1, n1: 64 values a wave, all twice
  auto load_bias = [&](int buf) __attribute__((always_inline)) {
    if (!a.bias) return;
    const long n0 = min(n1, a.n - 256);
    if (a.bias_f32)
      wide_load4((const float*)a.bias + n0, (tid & 255) * 4, lds_b + buf * kWideBias);
    else
      wide_load2((const bf16*)a.bias + n0, (tid & 255) * 2, lds_b + buf * kWideBias);
  };

  auto w_part = [&](int t, int buf) __attribute__((always_inline)) {
    const int row = wn * 128 + (t / 2) * 32 + (r / 4) * 8 + (t & 1) * 4 + (r & 3);
    return read_frag(all + buf * kWideW + row * 128, q, swizzle_w((r / 4) * 8 + (r & 3)));
  };
  auto x_part = [&](int u, int buf) __attribute__((always_inline)) {
    return read_frag(all + (2 + buf) * kWideW + ((wm * 4 + u) * 16 + r) * 128, q,
                     swizzle_x(r));
  };
  unsigned raw[5];  // the scales of four rows and of W, as they are held
  auto read_scales = [&](int buf) __attribute__((always_inline)) {
    const unsigned* const from = (const unsigned*)(all + 4 * kWideW + buf * kWideScales);
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = from[(wm * 4 + u) * 16 + r];
    raw[4] = from[256 + wn];
  };
  float s[4];
  auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      s[u] = both_scales(scale_value<SF>(raw[u]), scale_value<SF>(raw[4]));
  };

  enter();
  load_bias(0);
#pragma unroll
  for (int i = 0; i < 5; ++i) load_x(i, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) load_w(wfrom, i, 0);
  next();
#pragma unroll
  for (int i = 0; i < 5; ++i) load_x(i, 1);
  asm volatile("s_waitcnt vmcnt(5)\n\ts_barrier" ::: "memory");
  i32x8 xf[4], wf[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) xf[u] = x_part(u, 0);
  wf[0] = w_part(0, 0);
  wf[1] = w_part(1, 0);
  read_scales(0);
  take_scales();

  int buf = 0, tiles = 0, own_m = m1, own_n = n1;
  for (int tile = first; tile < end; tile += step) {
    float acc[8][4][4] = {};
    f32x4 p[4] = {};  // results of the last instructions
    float s_before = 0.f;  // the scale of the last two before this block
    for (int b = 0; b < kb; ++b) {
      // the rest of the next block, then the one after it
      const unsigned char* const wrest = wfrom;
      next();
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int j = i / 8, u = i % 8 / 2, t = 2 * j + i % 2;
        if (i == kTurn) stage_wait();
        if (i % 8 == 0) {
          const int from = i < kTurn ? buf : buf ^ 1, t2 = (2 * j + 2) % 8;
          wf[t2 % 4] = w_part(t2, from);
          wf[t2 % 4 + 1] = w_part(t2 + 1, from);
          if (i == kTurn) read_scales(buf ^ 1);
        }
        if (i > kTurn && i % 2 == 0) xf[u - 1] = x_part(u - 1, buf ^ 1);
        p[i % 4] = mfma128(wf[t % 4], xf[u]);
        const int o = (i + 30) % 32;  // the one whose result is there
        const float so = i < 2 ? s_before : s[o % 8 / 2];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[o / 8 * 2 + o % 2][o % 8 / 2][e] += p[o % 4][e] * so;
        if (i < 8 && i % 2 == 0) load_w(wrest, i / 2, buf ^ 1);
        if (i >= kTurn && i < kTurn + 5) load_x(i - kTurn, buf);
        __builtin_amdgcn_sched_barrier(0);  // in this order
      }
      xf[3] = x_part(3, buf ^ 1);
      s_before = s[3];
      take_scales();
      buf ^= 1;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[6 + h][3][e] += p[2 + h][e] * s_before;

    load_bias(~tiles & 1);
    // None of what follows is worked out ahead of the blocks.
    const int id = opaque(tid) & 63, re = id & 15, qe = id >> 4;
    const int m0 = min(own_m, a.m - 256), n0 = min(own_n, a.n - 256);
    const int nw = n0 + wn * 128;
    if (a.bias) {
      const unsigned* const bias =
          (const unsigned*)(all + 4 * kWideW + 2 * kWideScales +
                            (tiles & 1) * kWideBias) + wn * 128;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float b8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned v = bias[g * 32 + qe * 8 + i];
          b8[i] = a.bias_f32 ? __uint_as_float(v) : us2f((unsigned short)v);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[2 * g + i / 4][u][i & 3] += b8[i];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    ++tiles;
    if (a.gelu) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][u][i] = gelu<false>(acc[t][u][i]);
          __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (nw >= own_n) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = acc[i / 4][u][i & 3];
        const int m = m0 + (wm * 4 + u) * 16;
        // through shared memory, so that a store writes whole lines of 128 bytes: the
        // 8-bit rows at once, the others in two halves
        unsigned char* const out = all + kWideOut + wave * 2048;
        auto leave = [&](unsigned char* y, long pitch) __attribute__((always_inline)) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          uint4 line[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = i * 8 + id / 8, piece = id % 8;
            line[i] = *reinterpret_cast<const uint4*>(
                out + row * 128 + ((piece ^ (row & 7)) << 4));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (m + i * 8 + id / 8 >= own_m)
              store16_past(y + (m + i * 8 + id / 8) * pitch + id % 8 * 16, line[i]);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        };
        if (OUT == kBf16) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const float* const v8 = v + 16 * half + 8 * g;
              *reinterpret_cast<uint4*>(out + re * 128 + (((g * 4 + qe) ^ (re & 7)) << 4)) =
                  make_uint4(pack2_bf16(v8[0], v8[1]), pack2_bf16(v8[2], v8[3]),
                             pack2_bf16(v8[4], v8[5]), pack2_bf16(v8[6], v8[7]));
            }
            leave((unsigned char*)((bf16*)a.y + nw + half * 64), 2l * a.n);
          }
        } else {
          float most = absmax<32>(v);
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          const float scale = block_scale<SF>(most), inv = 1.0f / scale;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(out + re * 128 + (((g * 2 + qe / 2) ^ (re & 7)) << 4) +
                                      (qe & 1) * 8) = pack8_block(v + 8 * g, inv);
          if (qe == 0 && m + re >= own_m)
            store_scale<SF>(a.ys, (long)(m + re) * groups + nw / kBlock, scale);
          leave((unsigned char*)a.y + nw, a.n);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    own_m = m1;
    own_n = n1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was loaded past the last tile
}

template <Out OUT, bool SF>
void launch_wide(const GemmArgs& a, hipStream_t stream) {
  const int mtiles = ceil_div(a.m, 256), ntiles = ceil_div(a.n, 256);
  const long tiles = (long)mtiles * ntiles;
  const dim3 grid((unsigned)(tiles < 256 ? tiles : 256));
  hipLaunchKernelGGL((block_gemm_wide_kernel<OUT, SF>), grid, dim3(512), kWideLds, stream,
                     a, mtiles, ntiles);
}

template <int NT, int MT, Out OUT, bool SF>
void launch_direct(const GemmArgs& a, hipStream_t stream) {
  const dim3 grid(ceil_div(a.n, NT * 16) * ceil_div(a.m, 16 * MT));
  hipLaunchKernelGGL((block_gemm_direct_kernel<NT, MT, OUT, SF>), grid, dim3(512), 0,
                     stream, a);
}

// The larger the tile the less is read for each result, as long as every compute
// unit has a workgroup or two. us a call with bias to bf16, one call over and over in a
// graph ("x2": two teams):
//   rows x width x shared  direct 16x32  32x64  tiles 128x64 x2  128x64  128x128  256x128
//   38 x 768 x 768                  3.8    5.1              6.0     6.1      7.7     10.3
//   38 x 8192 x 4096               28     17               21      28       33       40
//   256 x 1601 x 1024              11      7.5              8.2     8.6     10.9     14.8
//   608 x 768 x 3072               25     16               14      17       22       29
//   1616 x 1601 x 1024             50     37               15      14       15       19
//   6464 x 3072 x 768                                      40      32       27       30
//   16384 x 1024 x 1024                                            32       29       26
//   103424 x 1024 x 1024                                          176      140      126
// Of few rows what counts is where W comes from. With other weights each call (60 MB of
// them), as in a model, instead of the caches:
//   38 x 8192 x 4096               29     18               21      28
//   256 x 1601 x 1024              11      7.7              9.1    10.3
//   608 x 768 x 1024               10      6.7              8.4     9.4
//   608 x 768 x 3072               23     13.8             16.8    20.6
//   1024 x 512 x 4096              32     18.6             20.1    25.8
// so that the direct kernel has them, also where two teams are faster in a loop.
//
// Tiles of 256 x 256 and the best of the others, by rounds of 256 tiles; one call over
// and over in a graph, to bf16 / to bf16 with GELU / to 8 bits / to 8 bits with GELU:
//   rows x width x shared   rounds  others                       256 x 256
//   9728 x 768 x 3072        0.45    36.3 / 37.4 / 35.1 / 37.6   40.8 / 43.6 / 40.0 / 44.0
//   12928 x 1024 x 1024      0.80    22.9 / 27.9 / 23.2 / 27.7   23.2 / 26.5 / 21.9 / 26.5
//   6464 x 3072 x 768        1.22    27.8 / 32.2 / 27.3 / 33.6   32.4 / 38.9 / 31.4 / 39.8
//   9728 x 3072 x 768        1.78    37.0 / 45.3 / 35.6 / 43.7   35.0 / 41.7 / 32.5 / 41.3
//   38912 x 768 x 3072       1.78    95.8 / 106 / 96.4 / 102     87.9 / 96.3 / 86.6 / 95.3
//   16384 x 4096 x 4096      4.00    269 / 292 / 276 / 284       237 / 249 / 238 / 257
//   103424 x 1024 x 1024     6.31    132 / 160 / 126 / 149       126 / 148 / 116 / 148
//   38912 x 3072 x 768       7.13    117 / 153 / 116 / 139       111 / 139 / 109 / 140
//   38912 x 3072 x 1536      7.13    208 / 234 / 202 / 227       195 / 219 / 186 / 220
// and to 8 bits with GELU, three sets of operands in turn, 103424 x 1024 x 1024 158 and
// 145, 25856 x 1024 x 1024 45 and 42, 51712 x 1024 x 512 56 and 57, 38912 x 3072 x 384
// 99 and 99; in the served encoder 162 and 149.
template <Out OUT, bool SF>
void launch_best(const GemmArgs& a, hipStream_t stream) {
  const int m = a.m, n = a.n, k = a.k;
  auto tiles = [&](long of_n, long of_m) {
    return ((n + of_n - 1) / of_n) * ((m + of_m - 1) / of_m);
  };
  constexpr long kUnits = 256;  // compute units
  if constexpr (OUT != kFp8) {
    if (tiles(16, 32) <= 2 * kUnits)
      return m <= 16 ? launch_direct<1, 1, OUT, SF>(a, stream)
                     : launch_direct<1, 2, OUT, SF>(a, stream);
    if (tiles(32, 64) <= kUnits) return launch_direct<2, 4, OUT, SF>(a, stream);
  }
  if (tiles(128, 64) <= kUnits) return launch_tiles<1, 4, 1, 2, OUT, SF>(a, stream);
  if (tiles(128, 64) <= 2 * kUnits) return launch_tiles<1, 4, 1, 1, OUT, SF>(a, stream);
  if constexpr (!kExact<OUT, SF>) {
    // 256 x 256 where workgroups come out about even
    const long wide = tiles(256, 256), rounds = (wide + kUnits - 1) / kUnits;
    if (k % kBlock == 0 && k >= 2 * kBlock && n % kBlock == 0 && n >= 256 && m >= 256 &&
        4 * wide >= 3 * rounds * kUnits)
      return launch_wide<OUT, SF>(a, stream);
    // 256 x 128 goes round twice a unit at a time: the last round has to be worth it
    const long large = tiles(256, 128), round = 2 * kUnits;
    if (large >= 4 * round || 10 * large >= 8 * ((large + round - 1) / round) * round)
      return launch_tiles<2, 2, 4, 1, OUT, SF>(a, stream);
  }
  // exact products too: 256 x 128 has no registers left for their operands. To f32 / to
  // 8 bits with f32 scales / the same with GELU, beside 8 bits with bf16 scales, us:
  //   38912 x 3072 x 768      243 / 188 / 240, 100
  //   103424 x 1024 x 1024    266 / 216 / 260, 113
  launch_tiles<1, 4, 2, 1, OUT, SF>(a, stream);
}

}  // namespace

// y in bf16, in f32 where y_f32, or in e4m3 where `ys` takes its scales. Scales, those
// of y as well, are bf16 or f32 as scales_f32 says.
void launch_block_gemm(const unsigned char* x, const void* xs, const unsigned char* w,
                       const void* ws, bool scales_f32, const void* bias, bool bias_f32,
                       void* y, bool y_f32, void* ys, long x_pitch, long w_pitch, int m,
                       int n, int k, bool gelu, hipStream_t stream) {
  const GemmArgs a{x,       w,       xs, ws, bias, y,    ys,
                   x_pitch, w_pitch, m,  n,  k,    gelu, bias_f32};
  if (ys)
    scales_f32 ? launch_best<kFp8, true>(a, stream) : launch_best<kFp8, false>(a, stream);
  else if (y_f32)
    scales_f32 ? launch_best<kF32, true>(a, stream) : launch_best<kF32, false>(a, stream);
  else
    scales_f32 ? launch_best<kBf16, true>(a, stream) : launch_best<kBf16, false>(a, stream);
}
