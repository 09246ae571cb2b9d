// Rotary position embedding of q and k heads: the pair (a, b) of frequency i, at position t, becomes
//
//   (a cos - b sin, b cos + a sin) * factor,   angle = t * inv_freq[i]
//
// with pairs (i, i + pairs) in the half layout, (2 i, 2 i + 1) interleaved; what lies past the 2 *
// pairs turned values of a head is copied. transposed turns by the negative angle: with the same
// factor, the gradient of the forward form.
//
// Angles: t * inv_freq in float64 (a float32 product is 0.004 radians off at position 100 000, as
// much as a bf16 rounding), reduced there to the nearest quarter turn and within it evaluated by
// the sine's and cosine's own power series in float32, to the last float32 bit or two.
#include <type_traits>

#include "block_fp8.h"
#include "sincos_turn.h"

namespace {

struct RotaryParams {
  const void* q;
  int64_t q_token, q_head;
  void* q_out;
  int64_t qo_token, qo_head;
  const void* k;
  int64_t k_token, k_head;
  void* k_out;
  int64_t ko_token, ko_head;
  const void* positions;
  int positions64;
  int64_t position_stride;
  const double* inv_freq;
  float factor;
  int negative;
  int64_t items;  // tokens * head groups * chunks
  int heads, all_heads, groups, pairs, dim, turned_chunks, chunks;
};

constexpr int kHeadsPerThread = 4;

// A thread turns V pairs of one frequency chunk of up to four heads of a token (or copies 2 V values
// past the turned ones), so that its sines and cosines serve all four. HBM bounds it where other waves
// hide a wave's latency: 16001 tokens of 40 heads of 128 in bf16 74 us, 4.4 TB/s (a copy 5.05); two
// heads a thread 82 us, eight 76. In few tokens its own chain does, 64 of 24 heads 6.2 us: each of the
// eight loads stands under a branch of load_values, through a pointer that is q's or k's, and is
// complete before the next goes out; the position and the frequencies follow them.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= p.items) return;
  const int64_t rest = item / p.chunks;
  const int chunk = (int)(item - rest * p.chunks);
  const int64_t token = rest / p.groups;
  const int head0 = (int)(rest - token * p.groups) * kHeadsPerThread;
  const bool turned = chunk < p.turned_chunks;
  // the chunk's two runs of V values, neighbours' runs side by side: in the half layout the pairs'
  // first and second values; interleaved (V > 1), V / 2 pairs of the first half of the pairs and as
  // many of the second; of what is copied, one run of each half (in turn where it has no halves)
  const int past = 2 * p.pairs, rest_dim = p.dim - past, copied = chunk - p.turned_chunks;
  const bool halves = rest_dim % (2 * V) == 0;
  const int at0 = turned ? chunk * (INTERLEAVED && V == 1 ? 2 : V) : past + copied * (halves ? V : 2 * V);
  const int at1 = turned ? (INTERLEAVED && V == 1 ? at0 + 1 : at0 + p.pairs)
                         : at0 + (halves ? rest_dim / 2 : V);
  const int64_t valid1 = p.dim - at1;  // a copied run may end with the head

  const T* src[kHeadsPerThread];
  T* dst[kHeadsPerThread];
  float a[kHeadsPerThread][V], b[kHeadsPerThread][V];
#pragma unroll
  for (int i = 0; i < kHeadsPerThread; ++i) {
    const int head = head0 + i < p.all_heads ? head0 + i : p.all_heads - 1;
    if (head < p.heads) {
      src[i] = static_cast<const T*>(p.q) + token * p.q_token + head * p.q_head;
      dst[i] = static_cast<T*>(p.q_out) + token * p.qo_token + head * p.qo_head;
    } else {
      src[i] = static_cast<const T*>(p.k) + token * p.k_token + (head - p.heads) * p.k_head;
      dst[i] = static_cast<T*>(p.k_out) + token * p.ko_token + (head - p.heads) * p.ko_head;
    }
    load_values(src[i] + at0, p.dim - at0, a[i]);
    load_values(src[i] + at1, valid1, b[i]);
  }
  if (turned) {
    const int64_t at = token * p.position_stride;
    const double position = p.positions64 ? (double)static_cast<const int64_t*>(p.positions)[at]
                                          : (double)static_cast<const int32_t*>(p.positions)[at];
    float s[V], c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = !INTERLEAVED || V == 1 ? chunk * V + v
                    : v < V / 2            ? chunk * (V / 2) + v
                                           : p.pairs / 2 + chunk * (V / 2) + v - V / 2;
      sincos_turn(position * p.inv_freq[i] * 0.15915494309189535, &s[v], &c[v]);
      s[v] *= p.negative ? -p.factor : p.factor;
      c[v] *= p.factor;
    }
#pragma unroll
    for (int i = 0; i < kHeadsPerThread; ++i) {
      float lo[V], hi[V];
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          // pair v of the chunk: values 2 v and 2 v + 1 of runs a then b
          const float e0 = 2 * v < V ? a[i][2 * v % V] : b[i][2 * v % V];
          const float e1 = 2 * v + 1 < V ? a[i][(2 * v + 1) % V] : b[i][(2 * v + 1) % V];
          const float r0 = __builtin_fmaf(e0, c[v], -(e1 * s[v]));
          const float r1 = __builtin_fmaf(e1, c[v], e0 * s[v]);
          if (2 * v < V) lo[2 * v % V] = r0; else hi[2 * v % V] = r0;
          if (2 * v + 1 < V) lo[(2 * v + 1) % V] = r1; else hi[(2 * v + 1) % V] = r1;
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          lo[v] = __builtin_fmaf(a[i][v], c[v], -(b[i][v] * s[v]));
          hi[v] = __builtin_fmaf(b[i][v], c[v], a[i][v] * s[v]);
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        a[i][v] = lo[v];
        b[i][v] = hi[v];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kHeadsPerThread; ++i) {
    if (head0 + i >= p.all_heads) break;
    store_values(dst[i] + at0, p.dim - at0, a[i]);
    store_values(dst[i] + at1, valid1, b[i]);
  }
}

template <typename T, int V>
int launch(const RotaryParams& p, bool interleaved, hipStream_t stream) {
  const int64_t workgroups = (p.items + 255) / 256;
  if (workgroups > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, V, true>), dim3((unsigned)workgroups), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((rotary_kernel<T, V, false>), dim3((unsigned)workgroups), dim3(256), 0, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

template <typename T>
int launch_pairs(RotaryParams p, int64_t tokens, bool interleaved, hipStream_t stream) {
  // V pairs a thread: the most of 8, 4, 2, 1 that divide the pairs
  const int v = p.pairs % 8 == 0 ? 8 : p.pairs % 4 == 0 ? 4 : p.pairs % 2 == 0 ? 2 : 1;
  p.turned_chunks = p.pairs / v;
  p.chunks = p.turned_chunks + (p.dim - 2 * p.pairs + 2 * v - 1) / (2 * v);
  p.groups = (p.all_heads + kHeadsPerThread - 1) / kHeadsPerThread;
  p.items = tokens * p.groups * p.chunks;
  switch (v) {
    case 8: return launch<T, 8>(p, interleaved, stream);
    case 4: return launch<T, 4>(p, interleaved, stream);
    case 2: return launch<T, 2>(p, interleaved, stream);
    default: return launch<T, 1>(p, interleaved, stream);
  }
}

}  // namespace

extern "C" int omni_rotary(const omni_rotary_args* a, omni_stream_t stream) {
  if (!a || a->tokens < 0 || a->heads < 1 || a->kv_heads < 0 || a->dim < 2 || a->pairs < 1 ||
      2 * a->pairs > a->dim || a->dim > 65536 || a->heads + a->kv_heads > 65536)
    return OMNI_ERR_INVALID_ARG;
  if (a->layout != OMNI_ROTARY_HALF && a->layout != OMNI_ROTARY_INTERLEAVED)
    return OMNI_ERR_INVALID_ARG;
  if (a->positions_dtype != OMNI_DTYPE_I32 && a->positions_dtype != OMNI_DTYPE_I64)
    return OMNI_ERR_INVALID_ARG;
  if (a->tokens == 0) return OMNI_OK;
  const int size = a->dtype == OMNI_DTYPE_F32 ? 4 : 2;
  if (!a->q || !a->q_out || !a->positions || !a->inv_freq ||
      (a->kv_heads > 0 && (!a->k || !a->k_out)) || !aligned_to(a->q, size) ||
      !aligned_to(a->q_out, size) || !aligned_to(a->k, size) || !aligned_to(a->k_out, size) ||
      !aligned_to(a->inv_freq, 8) ||
      !aligned_to(a->positions, a->positions_dtype == OMNI_DTYPE_I64 ? 8 : 4))
    return OMNI_ERR_INVALID_ARG;
  RotaryParams p{};
  p.q = a->q;
  p.q_token = a->q_stride_token;
  p.q_head = a->q_stride_head;
  p.q_out = a->q_out;
  p.qo_token = a->q_out_stride_token;
  p.qo_head = a->q_out_stride_head;
  p.k = a->k;
  p.k_token = a->k_stride_token;
  p.k_head = a->k_stride_head;
  p.k_out = a->k_out;
  p.ko_token = a->k_out_stride_token;
  p.ko_head = a->k_out_stride_head;
  p.positions = a->positions;
  p.positions64 = a->positions_dtype == OMNI_DTYPE_I64;
  p.position_stride = a->positions_stride;
  p.inv_freq = a->inv_freq;
  p.factor = a->factor;
  p.negative = a->transposed ? 1 : 0;
  p.heads = (int)a->heads;
  p.all_heads = (int)(a->heads + a->kv_heads);
  p.pairs = (int)a->pairs;
  p.dim = (int)a->dim;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool inter = a->layout == OMNI_ROTARY_INTERLEAVED;
  switch (a->dtype) {
    case OMNI_DTYPE_F32: return launch_pairs<float>(p, a->tokens, inter, s);
    case OMNI_DTYPE_BF16: return launch_pairs<__bf16>(p, a->tokens, inter, s);
    case OMNI_DTYPE_F16: return launch_pairs<_Float16>(p, a->tokens, inter, s);
    default: return OMNI_ERR_INVALID_ARG;
  }
}
