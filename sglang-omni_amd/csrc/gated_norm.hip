// The step between two blocks of a transformer, one pass over its rows:
//
//   u = post_norm(y)                       the block's output, normed (optional)
//   h = x + scale * act(gate) * u          the residual stream
//   n = pre_norm(h)                        the next block's input
//
// with RMSNorm (v / sqrt(mean(v^2) + eps) * weight) or LayerNorm ((v - mean) / sqrt(var + eps) *
// weight + bias) for both norms. n is formed from h before h is rounded to the stream's type.
//
// HBM bounds it: x, y and the gate are read once and h and n written once, a row staying in the
// registers of the 64, 256 or 1024 threads that hold it, 8 to 32 channels each, in float32; variances
// are sums of squared differences from the mean, formed after it. 16384 x 4096 in bf16, both norms, a
// gate per token: 127 us, 5.3 TB/s. Rows of up to 1024 channels are a wave's, without a barrier.
// With fewer rows, which do not hide it, the latency of a wave's own loads bounds it (3003 x 1000 10.5
// us, 2.4 TB/s; 1 x 1024 5.2 us): those of y and x stand under load_values' branches, each complete
// before the next goes out, and the weights, biases and the gate are loaded after the sums.
#include <type_traits>

#include "block_fp8.h"

namespace {

struct NormParams {
  const void* x;
  int64_t x_stride;
  const void* y;
  int64_t y_stride;
  const float* post_weight;
  const float* post_bias;
  const float* pre_weight;
  const float* pre_bias;
  const void* gate;
  int gate_dtype;
  int64_t gate_stride, rows_per_gate;
  int activation;
  float scale, eps;
  int post, layer;
  int64_t rows;
  int channels;
  void* h;
  int64_t h_stride;
  void* n;
  int n_dtype;
  int64_t n_stride;
  float* n_scale;
  int64_t n_scale_stride;
};

OMNI_DEVICE float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// The sum of v over the T threads of a row, in one fixed order. Each call takes LDS of its own, so
// one barrier is enough.
template <int T>
OMNI_DEVICE float row_sum(float v, float* lds) {
  v = wave_sum(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += lds[w];
  }
  return v;
}

template <int N>
OMNI_DEVICE void load_dtype(const void* src, int dtype, int64_t at, int64_t valid, float (&v)[N]) {
  if (dtype == OMNI_DTYPE_F32)
    load_values(static_cast<const float*>(src) + at, valid, v);
  else if (dtype == OMNI_DTYPE_BF16)
    load_values(static_cast<const __bf16*>(src) + at, valid, v);
  else
    load_values(static_cast<const _Float16*>(src) + at, valid, v);
}

OMNI_DEVICE float gate_value(int activation, float z) {
  if (activation == OMNI_GATE_SIGMOID) return 1.f / (1.f + __expf(-z));
  if (activation == OMNI_GATE_TANH) return tanhf(z);
  return z;
}

// v = norm(v) over a row held as NC chunks of 8 by T threads; elements past the row are zero and
// take no part in the statistics.
template <int T, int NC>
OMNI_DEVICE void norm_row(const NormParams& p, float (&v)[NC][8], const int (&valid)[NC], int c0,
                          const float* weight, const float* bias, float* lds) {
  const float c = (float)p.channels;
  if (p.layer) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += v[i][e];
    const float mean = row_sum<T>(sum, lds) / c;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = e < valid[i] ? v[i][e] - mean : 0.f;
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[i][e], v[i][e], ss);
  ss = row_sum<T>(ss, lds + T / 64);
  const float inv = 1.f / sqrtf(ss / c + p.eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int at = c0 + i * T * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] *= inv;
    if (weight) {
      float w[8];
      load_values(weight + at, valid[i], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= w[e];
    }
    if (bias) {
      float b[8];
      load_values(bias + at, valid[i], b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] += b[e];
    }
  }
}

// T threads per row, NC chunks of 8 channels per thread: chunk i holds channels (i T + thread) 8.
template <typename X, typename Y, int T, int NC>
__global__ void __launch_bounds__(T < 256 ? 256 : T) gated_norm_kernel(const NormParams p) {
  constexpr int ROWS = T < 256 ? 256 / T : 1;
  __shared__ float lds[T > 64 ? 4 * (T / 64) : 1];
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / T;
  if (T <= 64 && row >= p.rows) return;  // whole waves; with T > 64 a workgroup is one row
  const int c0 = (threadIdx.x % T) * 8;
  int valid[NC];
  float x[NC][8], u[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    valid[i] = p.channels - (c0 + i * T * 8);
    load_values(static_cast<const Y*>(p.y) + row * p.y_stride + c0 + i * T * 8, valid[i], u[i]);
    load_values(static_cast<const X*>(p.x) + row * p.x_stride + c0 + i * T * 8, valid[i], x[i]);
  }
  if (p.post) norm_row<T, NC>(p, u, valid, c0, p.post_weight, p.post_bias, lds);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (p.gate) {
      float g[8];
      load_dtype(p.gate, p.gate_dtype, (row / p.rows_per_gate) * p.gate_stride + c0 + i * T * 8,
                 valid[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[i][e] *= gate_value(p.activation, g[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = __builtin_fmaf(p.scale, u[i][e], x[i][e]);
    store_values(static_cast<X*>(p.h) + row * p.h_stride + c0 + i * T * 8, valid[i], x[i]);
  }
  norm_row<T, NC>(p, x, valid, c0, p.pre_weight, p.pre_bias, lds + 2 * (T / 64));
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * T * 8;
    const int64_t at = row * p.n_stride + c;
    if (p.n_dtype == OMNI_DTYPE_FP8_E4M3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = e < valid[i] ? x[i][e] : 0.f;
      u32x2 q;
      const float s = quantize_group(x[i], &q);
      if (c < (p.channels + 15) / 16 * 16)
        *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p.n) + at) = q;
      if (c % kBlock == 0 && valid[i] > 0) p.n_scale[row * p.n_scale_stride + c / kBlock] = s;
    } else if (p.n_dtype == OMNI_DTYPE_F32) {
      store_values(static_cast<float*>(p.n) + at, valid[i], x[i]);
    } else if (p.n_dtype == OMNI_DTYPE_BF16) {
      store_values(static_cast<__bf16*>(p.n) + at, valid[i], x[i]);
    } else {
      store_values(static_cast<_Float16*>(p.n) + at, valid[i], x[i]);
    }
  }
}

template <typename X, typename Y, int T, int NC>
int launch(const NormParams& p, hipStream_t stream) {
  constexpr int ROWS = T < 256 ? 256 / T : 1;
  const int64_t workgroups = (p.rows + ROWS - 1) / ROWS;
  if (workgroups > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((gated_norm_kernel<X, Y, T, NC>), dim3((unsigned)workgroups),
                     dim3(T < 256 ? 256 : T), 0, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

template <typename X, typename Y>
int launch_width(const NormParams& p, hipStream_t stream) {
  const int c = p.channels;
  if (c <= 64 * 8) return launch<X, Y, 64, 1>(p, stream);
  if (c <= 64 * 16) return launch<X, Y, 64, 2>(p, stream);
  if (c <= 256 * 8) return launch<X, Y, 256, 1>(p, stream);
  if (c <= 256 * 16) return launch<X, Y, 256, 2>(p, stream);
  if (c <= 256 * 32) return launch<X, Y, 256, 4>(p, stream);
  if (c <= 1024 * 16) return launch<X, Y, 1024, 2>(p, stream);
  return launch<X, Y, 1024, 4>(p, stream);
}

bool float_dtype(int d) {
  return d == OMNI_DTYPE_F32 || d == OMNI_DTYPE_BF16 || d == OMNI_DTYPE_F16;
}

int size_of(int dtype) {
  return dtype == OMNI_DTYPE_F32 ? 4 : dtype == OMNI_DTYPE_FP8_E4M3 ? 1 : 2;
}

}  // namespace

extern "C" int omni_gated_residual_norm(const omni_gated_norm_args* a, omni_stream_t stream) {
  constexpr int kMaxChannels = 1024 * 32;
  if (!a || a->rows < 0 || a->channels < 1) return OMNI_ERR_INVALID_ARG;
  if (a->channels > kMaxChannels) return OMNI_ERR_UNSUPPORTED;
  if (a->rows == 0) return OMNI_OK;
  const bool fp8 = a->normed_dtype == OMNI_DTYPE_FP8_E4M3;
  if (!float_dtype(a->x_dtype) || !float_dtype(a->y_dtype) ||
      !(fp8 || float_dtype(a->normed_dtype)) || (a->gate && !float_dtype(a->gate_dtype)))
    return OMNI_ERR_INVALID_ARG;
  if (a->x_dtype != a->y_dtype && a->x_dtype != OMNI_DTYPE_F32) return OMNI_ERR_UNSUPPORTED;
  if ((a->norm != OMNI_NORM_RMS && a->norm != OMNI_NORM_LAYER) ||
      (a->gate_activation != OMNI_GATE_NONE && a->gate_activation != OMNI_GATE_SIGMOID &&
       a->gate_activation != OMNI_GATE_TANH) || !(a->eps >= 0.f))
    return OMNI_ERR_INVALID_ARG;
  if (a->norm == OMNI_NORM_RMS && (a->post_bias || a->pre_bias)) return OMNI_ERR_INVALID_ARG;
  const int64_t c = a->channels, padded = (c + 15) / 16 * 16;
  if (!a->x || !a->y || !a->residual || !a->normed || a->x_stride < c || a->y_stride < c ||
      a->residual_stride < c || a->normed_stride < (fp8 ? padded : c) ||
      (a->gate && (a->gate_stride < 0 || a->rows_per_gate < 1)))
    return OMNI_ERR_INVALID_ARG;
  if (!aligned_to(a->x, size_of(a->x_dtype)) || !aligned_to(a->y, size_of(a->y_dtype)) ||
      !aligned_to(a->residual, size_of(a->x_dtype)) ||
      !aligned_to(a->normed, fp8 ? 16 : size_of(a->normed_dtype)) ||
      (a->gate && !aligned_to(a->gate, size_of(a->gate_dtype))) || !aligned_to(a->post_weight, 4) ||
      !aligned_to(a->post_bias, 4) || !aligned_to(a->pre_weight, 4) || !aligned_to(a->pre_bias, 4))
    return OMNI_ERR_INVALID_ARG;
  if (fp8 && (!a->normed_scale || !aligned_to(a->normed_scale, 4) || a->normed_stride % 16 ||
              a->normed_scale_stride < (c + kBlock - 1) / kBlock))
    return OMNI_ERR_INVALID_ARG;
  NormParams p{};
  p.x = a->x;
  p.x_stride = a->x_stride;
  p.y = a->y;
  p.y_stride = a->y_stride;
  p.post_weight = a->post_weight;
  p.post_bias = a->post_bias;
  p.pre_weight = a->pre_weight;
  p.pre_bias = a->pre_bias;
  p.gate = a->gate;
  p.gate_dtype = a->gate_dtype;
  p.gate_stride = a->gate_stride;
  p.rows_per_gate = a->rows_per_gate;
  p.activation = a->gate_activation;
  p.scale = a->scale;
  p.eps = a->eps;
  p.post = a->post_norm ? 1 : 0;
  p.layer = a->norm == OMNI_NORM_LAYER ? 1 : 0;
  p.rows = a->rows;
  p.channels = (int)c;
  p.h = a->residual;
  p.h_stride = a->residual_stride;
  p.n = a->normed;
  p.n_dtype = a->normed_dtype;
  p.n_stride = a->normed_stride;
  p.n_scale = a->normed_scale;
  p.n_scale_stride = a->normed_scale_stride;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->y_dtype == OMNI_DTYPE_F32) return launch_width<float, float>(p, s);
  if (a->y_dtype == OMNI_DTYPE_BF16)
    return a->x_dtype == OMNI_DTYPE_F32 ? launch_width<float, __bf16>(p, s)
                                        : launch_width<__bf16, __bf16>(p, s);
  return a->x_dtype == OMNI_DTYPE_F32 ? launch_width<float, _Float16>(p, s)
                                      : launch_width<_Float16, _Float16>(p, s);
}
