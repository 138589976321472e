// Producers of block-scaled 8-bit rows, and the root-mean-square norm.
//
// All of it is bound by memory: each row is read once into registers, and what
// the row yields (the residual stream, the norm, its 8-bit form and scales) is
// written from there. A lane holds 8 neighbouring values, so one block of 128
// is 16 lanes of a wave and its largest value four exchanges away; a row is
// held by 16 or 32 lanes, by one wave, by four, or by sixteen, whichever keeps
// its values in registers and leaves few lanes idle.

#include "block_fp8.h"

namespace {

// sum over the L lanes that hold a row
template <int L>
DEV float row_sum(float v, float* lds) {
#pragma unroll
  for (int off = (L < WAVE ? L : WAVE) / 2; off; off >>= 1) v += __shfl_xor(v, off);
  if (L <= WAVE) return v;
  __syncthreads();  // the sums before these have been read
  if (lane_id() == 0) lds[wave_id()] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < L / WAVE; ++i) v += lds[i];
  return v;
}
constexpr int threads_of(int L) { return L <= WAVE ? 256 : L; }

enum Form { kRms, kRms8, kLayer8 };

template <typename T>
struct NormArgs {
  const T *x, *res, *w, *b;
  T *y, *sum;
  unsigned char* y8;
  void* scales;  // f32 by the kernels that are SF, else bf16
  float* rstd;
  long rows;
  int dim;
  float eps;
};

// us for 103424 rows of 1024 in bf16 (TB/s of what has to be moved): rms with the
// residual to 8 bits 135 (5.5), layer to both 111 (4.8), rms 78 (5.4); a copy of
// 2 GiB runs at 4.8.
//
// t = x + res; rms: y = t / sqrt(mean t^2 + eps) * w with t as the type holds
// it (it is the stream that goes on), layer: y = (t - mean) / sqrt(var + eps)
// * w + b with t in 32 bits.
//
// The type of the scales is the kernel's (SF): asked for at run time it takes six
// registers, and the layer norm of 1024 one wave less a SIMD (111 us became 113).
template <typename T, Form FORM, bool RES, bool SF, int L, int R>
__global__ __launch_bounds__(threads_of(L)) void block_norm_kernel(
    NormArgs<T> a) {
  constexpr int kRowsPerBlock = threads_of(L) / L;
  __shared__ float lds[16];
  const int t = threadIdx.x % L;
  const int dim = a.dim;
  const int groups = ceil_div(dim, kBlock);
  const long pitch = fp8_pitch(dim);
  const float inv_dim = 1.0f / dim;

  for (long row = (long)blockIdx.x * kRowsPerBlock + threadIdx.x / L;
       row < a.rows; row += (long)gridDim.x * kRowsPerBlock) {
    float v[R][8];
    float sq = 0.f, s = 0.f;
#pragma unroll
    for (int c = 0; c < R; ++c) {
      const int j = (c * L + t) * 8;
      load8_row(a.x + row * dim, j, dim, v[c]);
      if (RES) {
        float r8[8];
        load8_row(a.res + row * dim, j, dim, r8);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[c][i] += r8[i];
          if (FORM != kLayer8) v[c][i] = held(v[c][i], a.x);
        }
        if (FORM != kLayer8) store8_row(a.sum + row * dim, j, dim, v[c]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sq += v[c][i] * v[c][i];
        s += v[c][i];
      }
    }
    float rstd;
    if (FORM == kLayer8) {
      // the variance from the differences, which stay in registers
      const float mean = row_sum<L>(s, lds) * inv_dim;
      sq = 0.f;
#pragma unroll
      for (int c = 0; c < R; ++c) {
        const int j = (c * L + t) * 8;
        if (j + 8 <= dim) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] -= mean;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] = j + i < dim ? v[c][i] - mean : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += v[c][i] * v[c][i];
      }
    }
    rstd = rsqrtf(row_sum<L>(sq, lds) * inv_dim + a.eps);
    if (FORM == kRms && a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < R; ++c) {
      const int j = (c * L + t) * 8;
      float w8[8], y[8];
      load8_row(a.w, j, dim, w8);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[c][i] * rstd * w8[i];
      if (FORM == kLayer8) {
        float b8[8];
        load8_row(a.b, j, dim, b8);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] += b8[i];
      }
      if (FORM != kRms8) store8_row(a.y + row * dim, j, dim, y);
      if (FORM != kRms) {
        const float scale = block_scale<SF>(group16_max(absmax<8>(y)));
        if (j < dim) {
          *reinterpret_cast<uint2*>(a.y8 + row * pitch + j) =
              pack8_block(y, 1.0f / scale);
          if ((t & 15) == 0)
            store_scale<SF>(a.scales, row * groups + j / kBlock, scale);
        }
      }
    }
  }
}

// rows in blocks of 128: 16 lanes a block, no block needs another (103424 rows of
// 1024 in bf16: 59 us, 5.4 TB/s)
template <typename T, bool SF>
__global__ __launch_bounds__(256) void quantize_block_kernel(
    const T* __restrict__ x, unsigned char* __restrict__ y8,
    void* __restrict__ scales, long rows, int dim) {
  const int groups = ceil_div(dim, kBlock);
  const long pitch = fp8_pitch(dim);
  const long n = rows * groups;
  for (long g = (long)blockIdx.x * 16 + (threadIdx.x >> 4); g < n;
       g += (long)gridDim.x * 16) {
    const long row = g / groups;
    const int j = (int)(g - row * groups) * kBlock + (threadIdx.x & 15) * 8;
    float v[8];
    load8_row(x + row * dim, j, dim, v);
    const float scale = block_scale<SF>(group16_max(absmax<8>(v)));
    if (j < dim)
      *reinterpret_cast<uint2*>(y8 + row * pitch + j) = pack8_block(v, 1.0f / scale);
    if ((threadIdx.x & 15) == 0) store_scale<SF>(scales, g, scale);
  }
}

// a weight in blocks of 128 x 128: a workgroup a block, 8 rows of 16 values a
// thread's share, held in registers between the two passes
template <typename T, bool SF>
__global__ __launch_bounds__(256) void quantize_block_weight_kernel(
    const T* __restrict__ w, unsigned char* __restrict__ w8,
    void* __restrict__ scales, int n, int k) {
  __shared__ float lds[4];
  const long pitch = fp8_pitch(k);
  const int j = blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
  const int row0 = blockIdx.y * kBlock + (threadIdx.x >> 4);
  float v[8][8];
  float a = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int row = row0 + r * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[r][i] = 0.f;
    if (row < n) load8_row(w + (long)row * k, j, k, v[r]);
    a = fmaxf(a, absmax<8>(v[r]));
  }
  a = wave_max(a);
  if (lane_id() == 0) lds[wave_id()] = a;
  __syncthreads();
  const float scale =
      block_scale<SF>(fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3])));
  const float inv = 1.0f / scale;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int row = row0 + r * 16;
    if (row < n && j < k)
      *reinterpret_cast<uint2*>(w8 + row * pitch + j) = pack8_block(v[r], inv);
  }
  if (threadIdx.x == 0)
    store_scale<SF>(scales, (long)blockIdx.y * gridDim.x + blockIdx.x, scale);
}

// Backward of y = n * w, n = t * rstd:  h = gy * w,  c = mean(h * n),
//   gt = rstd * (h - n * c) + gsum,   gw = sum over rows of gy * n.
// A lane keeps the same columns for every row that its wave takes, so the
// weight's gradient adds up in registers; each workgroup writes one row of
// partial sums, which rms_weight_grad_kernel adds in a fixed order.
template <typename T, bool GSUM, int L, int R>
__global__ __launch_bounds__(threads_of(L)) void rms_bwd_kernel(
    const T* __restrict__ gy, const T* __restrict__ gsum,
    const T* __restrict__ t_in, const float* __restrict__ rstd_in,
    const T* __restrict__ w, T* __restrict__ gx, float* __restrict__ part,
    long rows, int dim) {
  constexpr int kRowsPerBlock = threads_of(L) / L;
  __shared__ float lds[16];
  __shared__ float all[L <= WAVE ? R * L * 8 : 1];
  const int t = threadIdx.x % L;
  float w8[R][8], gw[R][8];
#pragma unroll
  for (int c = 0; c < R; ++c) {
    load8_row(w, (c * L + t) * 8, dim, w8[c]);
#pragma unroll
    for (int i = 0; i < 8; ++i) gw[c][i] = 0.f;
  }
  for (long row = (long)blockIdx.x * kRowsPerBlock + threadIdx.x / L;
       row < rows; row += (long)gridDim.x * kRowsPerBlock) {
    const float rstd = rstd_in[row];
    float h[R][8], n[R][8];
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < R; ++c) {
      const int j = (c * L + t) * 8;
      load8_row(gy + row * dim, j, dim, h[c]);
      load8_row(t_in + row * dim, j, dim, n[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[c][i] *= rstd;
        gw[c][i] += h[c][i] * n[c][i];
        h[c][i] *= w8[c][i];
        dot += h[c][i] * n[c][i];
      }
    }
    const float mean = row_sum<L>(dot, lds) / dim;
#pragma unroll
    for (int c = 0; c < R; ++c) {
      const int j = (c * L + t) * 8;
      float g[8];
      if (GSUM) load8_row(gsum + row * dim, j, dim, g);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        g[i] = (GSUM ? g[i] : 0.f) + rstd * (h[c][i] - n[c][i] * mean);
      store8_row(gx + row * dim, j, dim, g);
    }
  }
  if (L <= WAVE) {
    // the rows' sums, in their order
    for (int k = 0; k < kRowsPerBlock; ++k) {
      if (threadIdx.x / L == k) {
#pragma unroll
        for (int c = 0; c < R; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float& at = all[(c * L + t) * 8 + i];
            at = k ? at + gw[c][i] : gw[c][i];
          }
      }
      __syncthreads();
    }
    for (int j = threadIdx.x; j < dim; j += 256)
      part[(long)blockIdx.x * dim + j] = all[j];
  } else {
#pragma unroll
    for (int c = 0; c < R; ++c)
      store8_row(part + (long)blockIdx.x * dim, (c * L + t) * 8, dim, gw[c]);
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void rms_weight_grad_kernel(
    const float* __restrict__ part, T* __restrict__ gw, int parts, int dim) {
  __shared__ float lds[16][WAVE];
  const int j = blockIdx.x * WAVE + lane_id();
  float s = 0.f;
  if (j < dim) {
    int p = wave_id();
    for (; p + 112 < parts; p += 128) {  // eight reads on their way at a time
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part[(long)(p + 16 * i) * dim + j];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; p < parts; p += 16) s += part[(long)p * dim + j];
  }
  lds[wave_id()][lane_id()] = s;
  __syncthreads();
  if (wave_id() == 0 && j < dim) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][lane_id()];
    st1(gw + j, s);
  }
}

constexpr int kUnits = 256;  // compute units

// rows that a workgroup holds at a time
int rows_at_once(int dim) {
  return dim <= 128 ? 16 : dim <= 256 ? 8 : dim <= 2048 ? 4 : 1;
}

template <typename T, Form FORM, bool RES, bool SF, int L, int R>
void norm_launch(const NormArgs<T>& a, hipStream_t stream) {
  constexpr int rows = threads_of(L) / L;
  const long blocks = (a.rows + rows - 1) / rows;
  // a launch has fewer than 2^32 threads
  const int grid = (int)(blocks < (1 << 21) ? blocks : (1 << 21));
  hipLaunchKernelGGL((block_norm_kernel<T, FORM, RES, SF, L, R>), dim3(grid),
                     dim3(threads_of(L)), 0, stream, a);
}

// the fewest lanes that hold a row in at most 32 values each, so that what a
// row needs stays in registers beside its weights; 64 a lane at the very end
#define BY_WIDTH(dim, LAUNCH)               \
  do {                                      \
    if (dim <= 128) LAUNCH(16, 1);          \
    else if (dim <= 256) LAUNCH(32, 1);     \
    else if (dim <= 512) LAUNCH(64, 1);     \
    else if (dim <= 1024) LAUNCH(64, 2);    \
    else if (dim <= 2048) LAUNCH(64, 4);    \
    else if (dim <= 4096) LAUNCH(256, 2);   \
    else if (dim <= 8192) LAUNCH(256, 4);   \
    else if (dim <= 16384) LAUNCH(1024, 2); \
    else if (dim <= 32768) LAUNCH(1024, 4); \
    else LAUNCH(1024, 8);                   \
  } while (0)

template <typename T, Form FORM, bool RES, bool SF>
void norm_by_width(const NormArgs<T>& a, hipStream_t stream) {
#define LAUNCH(L, R) norm_launch<T, FORM, RES, SF, L, R>(a, stream)
  BY_WIDTH(a.dim, LAUNCH);
#undef LAUNCH
}
template <typename T, Form FORM>
void norm_by_kind(const NormArgs<T>& a, bool scales_f32, hipStream_t stream) {
  if constexpr (FORM != kRms) {
    if (scales_f32)
      return a.res ? norm_by_width<T, FORM, true, true>(a, stream)
                   : norm_by_width<T, FORM, false, true>(a, stream);
  }
  a.res ? norm_by_width<T, FORM, true, false>(a, stream)
        : norm_by_width<T, FORM, false, false>(a, stream);
}

}  // namespace

// form 0: y (and rstd where it is given); 1: y8 and scales; 2: layer norm, y,
// y8 and scales. `sum` is written by forms 0 and 1 where `res` is given.
template <typename T>
void launch_block_norm(int form, const T* x, const T* res, const T* w,
                       const T* b, T* y, T* sum, unsigned char* y8,
                       void* scales, bool scales_f32, float* rstd, long rows,
                       int dim, float eps, hipStream_t stream) {
  const NormArgs<T> a{x, res, w, b, y, sum, y8, scales, rstd, rows, dim, eps};
  if (form == 0)
    norm_by_kind<T, kRms>(a, scales_f32, stream);
  else if (form == 1)
    norm_by_kind<T, kRms8>(a, scales_f32, stream);
  else
    norm_by_kind<T, kLayer8>(a, scales_f32, stream);
}

// How many rows of partial sums launch_rms_bwd writes: four workgroups a compute
// unit where a workgroup holds several rows (103424x1024 bf16: 112 us, with two of
// them 163, with eight 114 and twice as long to add up), two where it holds one.
int rms_bwd_parts(long rows, int dim) {
  const int at_once = rows_at_once(dim);
  const long blocks = (rows + at_once - 1) / at_once;
  const long most = (at_once > 1 ? 4 : 2) * kUnits;
  return (int)(blocks < most ? blocks : most);
}

template <typename T>
void launch_rms_bwd(const T* gy, const T* gsum, const T* t, const float* rstd,
                    const T* w, T* gx, T* gw, float* part, long rows, int dim,
                    hipStream_t stream) {
  const int parts = rms_bwd_parts(rows, dim);
#define LAUNCH(L, R)                                                          \
  do {                                                                        \
    if (gsum)                                                                 \
      hipLaunchKernelGGL((rms_bwd_kernel<T, true, L, R>), dim3(parts),        \
                         dim3(threads_of(L)), 0, stream, gy,                  \
                         gsum, t, rstd, w, gx, part, rows, dim);              \
    else                                                                      \
      hipLaunchKernelGGL((rms_bwd_kernel<T, false, L, R>), dim3(parts),       \
                         dim3(threads_of(L)), 0, stream, gy,                  \
                         gsum, t, rstd, w, gx, part, rows, dim);              \
  } while (0)
  BY_WIDTH(dim, LAUNCH);
#undef LAUNCH
  hipLaunchKernelGGL((rms_weight_grad_kernel<T>), dim3(ceil_div(dim, WAVE)),
                     dim3(1024), 0, stream, part, gw, parts, dim);
}

template <typename T>
void launch_quantize_block(const T* x, unsigned char* y8, void* scales,
                           bool scales_f32, long rows, int dim,
                           hipStream_t stream) {
  const long blocks = (rows * ceil_div(dim, kBlock) + 15) / 16;
  const dim3 grid((int)(blocks < 8192 ? blocks : 8192));
  if (scales_f32)
    hipLaunchKernelGGL((quantize_block_kernel<T, true>), grid, dim3(256), 0, stream, x,
                       y8, scales, rows, dim);
  else
    hipLaunchKernelGGL((quantize_block_kernel<T, false>), grid, dim3(256), 0, stream, x,
                       y8, scales, rows, dim);
}

template <typename T>
void launch_quantize_block_weight(const T* w, unsigned char* w8, void* scales,
                                  bool scales_f32, int n, int k,
                                  hipStream_t stream) {
  const dim3 grid(ceil_div(k, kBlock), ceil_div(n, kBlock));
  if (scales_f32)
    hipLaunchKernelGGL((quantize_block_weight_kernel<T, true>), grid, dim3(256), 0,
                       stream, w, w8, scales, n, k);
  else
    hipLaunchKernelGGL((quantize_block_weight_kernel<T, false>), grid, dim3(256), 0,
                       stream, w, w8, scales, n, k);
}

#define INSTANTIATE(T)                                                        \
  template void launch_block_norm<T>(int, const T*, const T*, const T*,       \
                                     const T*, T*, T*, unsigned char*,        \
                                     void*, bool, float*, long, int, float,   \
                                     hipStream_t);                            \
  template void launch_rms_bwd<T>(const T*, const T*, const T*, const float*, \
                                  const T*, T*, T*, float*, long, int,        \
                                  hipStream_t);                               \
  template void launch_quantize_block<T>(const T*, unsigned char*, void*,     \
                                         bool, long, int, hipStream_t);       \
  template void launch_quantize_block_weight<T>(                              \
      const T*, unsigned char*, void*, bool, int, int, hipStream_t);
INSTANTIATE(bf16)
INSTANTIATE(float)
