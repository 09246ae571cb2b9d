// The heads of a transformer layer between its qkv product and its attention, in one launch:
//
//   q, k heads   n = x / sqrt(mean(x^2) + eps) * weight        (RMS over the head; omitted for rows
//                                                              that are only written)
//                then rotary positions: the pair (a, b) of frequency i becomes
//                (a cos - b sin, b cos + a sin) * factor, angle = position * inv_freq[i]
//   k, v heads   into the paged cache's row of the token's slot, as they are or in E4M3 with a scale
//                per row, scale = amax / 448
//
// and the way back: rows of the cache by slot. Angles in float64 as in the rotary kernel; everything
// else in float32, rounded once to the rows' type; what the cache gets is that rounded value, so one
// launch leaves the bits of norm, rotation and write one after the other.
//
// Each value is read and written once, so HBM bounds long prompts: 16001 tokens of 32 + 8 heads of 128 in
// bf16 69 us, 4.7 TB/s (a copy 5.06), and with the keys and values into an 8-bit cache 100; 30011 rows of 8
// to 8 bits 40 - 45 and back 33. A decode step is one chain of loads (rows, weights, position and frequencies
// together, then the slot) and its reductions: 64 tokens of 16 + 8 heads into the cache 4.3 us in a graph (4.9
// in 8 bits), 5.8 where the GPU is waited for after each.
#include <type_traits>

#include "kv_cache.h"
#include "sincos_turn.h"

namespace {

struct HeadsParams {
  const void* src[3];  // q, k, v
  int64_t src_token[3], src_head[3];
  void* dst[2];  // q, k; null: not wanted
  int64_t dst_token[2], dst_head[2];
  const float* weight[2];
  const void* positions;
  int positions64;
  int64_t position_stride;
  const double* inv_freq;
  float factor, eps;
  int normed, interleaved;
  CacheView cache;
  int held;  // the cache's type, -1: no cache
  const void* slots;
  int slots64;
  int64_t slots_stride;
  int64_t items;  // tokens * groups
  int heads[3], groups[3];
  int pairs, dim, turned_chunks, chunks, lane_shift;
};

OMNI_DEVICE int64_t load_index(const void* p, int wide, int64_t at) {
  return wide ? static_cast<const int64_t*>(p)[at] : (int64_t) static_cast<const int32_t*>(p)[at];
}

// The float32 value of v rounded to T.
template <typename T>
OMNI_DEVICE float rounded(float v) {
  return (float)(T)v;
}

// V values as E4M3 bytes at dst, those below `valid` alone.
template <int V>
OMNI_DEVICE void store_bytes(uint8_t* dst, int valid, const float (&v)[V], float unit) {
  uint8_t bytes[V];
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[i] * unit, (i + 1 < V ? v[(i + 1) % V] : 0.f) * unit,
                                                  0, false);
    bytes[i] = (uint8_t)w;
    if (i + 1 < V) bytes[(i + 1) % V] = (uint8_t)(w >> 8);
  }
  if (valid >= V) {
    __builtin_memcpy(dst, bytes, V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) dst[i] = bytes[i];
  }
}

// 2^lane_shift lanes take HP heads of one kind (q, k or v) of a token. A lane holds of each head ITERS
// chunks of two runs of V values: in the half layout V pairs' first and second values, interleaved V /
// 2 pairs of the first half of the pairs and as many of the second; of what is not turned one run of
// each half (in turn where it has no halves). A chunk's sines and cosines serve all HP heads.
//
// WHOLE: every run of a chunk lies in the head. Then a lane's loads, of rows, weights, position and
// frequencies, have no branch around them and go out at once (a load under a branch is waited for before
// the next one goes out); lanes past the last chunk load it too, are not turned, and count nothing: neither
// in the sum of squares nor in an 8-bit row's largest magnitude.
template <typename T, int V, int ITERS, int HP, bool WHOLE>
__global__ void __launch_bounds__(256) heads_kernel(const HeadsParams p) {
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> p.lane_shift;
  if (item >= p.items) return;
  const int lanes = 1 << p.lane_shift, lane = threadIdx.x & (lanes - 1);
  const int all_groups = p.groups[0] + p.groups[1] + p.groups[2];
  const int64_t token = item / all_groups;
  int group = (int)(item - token * all_groups), kind = 0;
  if (group >= p.groups[0]) {
    group -= p.groups[0];
    kind = 1;
    if (group >= p.groups[1]) {
      group -= p.groups[1];
      kind = 2;
    }
  }
  const int heads = kind == 0 ? p.heads[0] : kind == 1 ? p.heads[1] : p.heads[2];
  const T* src = static_cast<const T*>(kind == 0 ? p.src[0] : kind == 1 ? p.src[1] : p.src[2]) +
                 token * (kind == 0 ? p.src_token[0] : kind == 1 ? p.src_token[1] : p.src_token[2]);
  const int64_t src_head = kind == 0 ? p.src_head[0] : kind == 1 ? p.src_head[1] : p.src_head[2];
  const int head0 = group * HP;

  int at0[ITERS], at1[ITERS], valid0[ITERS], valid1[ITERS];
  const int past = 2 * p.pairs, rest = p.dim - past;
  const bool halves = rest % (2 * V) == 0;
  const bool single = V == 1 && p.interleaved;
#pragma unroll
  for (int t = 0; t < ITERS; ++t) {
    const int mine = lane + t * lanes, chunk = WHOLE && mine >= p.chunks ? p.chunks - 1 : mine;
    const int copied = chunk - p.turned_chunks;
    const bool turned = chunk < p.turned_chunks;
    at0[t] = turned ? chunk * (single ? 2 : V) : past + copied * (halves ? V : 2 * V);
    at1[t] = turned ? (single ? at0[t] + 1 : at0[t] + p.pairs) : at0[t] + (halves ? rest / 2 : V);
    valid0[t] = mine < p.chunks ? p.dim - at0[t] : 0;
    valid1[t] = mine < p.chunks ? p.dim - at1[t] : 0;
  }
  double position = 0.0;
  if (p.pairs > 0) position = (double)load_index(p.positions, p.positions64, token * p.position_stride);

  float a[HP][ITERS][V], b[HP][ITERS][V];
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    const T* row = src + (head0 + i < heads ? head0 + i : heads - 1) * src_head;
#pragma unroll
    for (int t = 0; t < ITERS; ++t) {
      load_values(row + at0[t], WHOLE ? V : valid0[t], a[i][t]);
      load_values(row + at1[t], WHOLE ? V : valid1[t], b[i][t]);
    }
  }
  if (p.normed && kind < 2) {
    const float* weight = kind == 0 ? p.weight[0] : p.weight[1];
    float w0[ITERS][V], w1[ITERS][V];
#pragma unroll
    for (int t = 0; t < ITERS; ++t) {
      if (weight) {
        load_values(weight + at0[t], WHOLE ? V : valid0[t], w0[t]);
        load_values(weight + at1[t], WHOLE ? V : valid1[t], w1[t]);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) w0[t][v] = w1[t][v] = 1.f;
      }
    }
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < ITERS; ++t) {
        float part = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
          part = __builtin_fmaf(a[i][t][v], a[i][t][v], __builtin_fmaf(b[i][t][v], b[i][t][v], part));
        sum += WHOLE && valid0[t] == 0 ? 0.f : part;
      }
      for (int off = 1; off < lanes; off <<= 1) sum += __shfl_xor(sum, off);
      const float r = 1.f / sqrtf(sum / (float)p.dim + p.eps);
#pragma unroll
      for (int t = 0; t < ITERS; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          a[i][t][v] *= r * w0[t][v];
          b[i][t][v] *= r * w1[t][v];
        }
    }
  }
  if (p.pairs > 0 && kind < 2) {
#pragma unroll
    for (int t = 0; t < ITERS; ++t) {
      const int chunk = lane + t * lanes;
      if (chunk >= p.turned_chunks) continue;
      float s[V], c[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = !p.interleaved || V == 1 ? chunk * V + v
                      : v < V / 2              ? chunk * (V / 2) + v
                                               : p.pairs / 2 + chunk * (V / 2) + v - V / 2;
        sincos_turn(position * p.inv_freq[i] * 0.15915494309189535, &s[v], &c[v]);
        s[v] *= p.factor;
        c[v] *= p.factor;
      }
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        float lo[V], hi[V];
        if (p.interleaved && V > 1) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            // pair v of the chunk: values 2 v and 2 v + 1 of runs a then b
            const float e0 = 2 * v < V ? a[i][t][2 * v % V] : b[i][t][2 * v % V];
            const float e1 = 2 * v + 1 < V ? a[i][t][(2 * v + 1) % V] : b[i][t][(2 * v + 1) % V];
            const float r0 = __builtin_fmaf(e0, c[v], -(e1 * s[v]));
            const float r1 = __builtin_fmaf(e1, c[v], e0 * s[v]);
            if (2 * v < V) lo[2 * v % V] = r0; else hi[2 * v % V] = r0;
            if (2 * v + 1 < V) lo[(2 * v + 1) % V] = r1; else hi[(2 * v + 1) % V] = r1;
          }
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            lo[v] = __builtin_fmaf(a[i][t][v], c[v], -(b[i][t][v] * s[v]));
            hi[v] = __builtin_fmaf(b[i][t][v], c[v], a[i][t][v] * s[v]);
          }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          a[i][t][v] = lo[v];
          b[i][t][v] = hi[v];
        }
      }
    }
  }
  if (kind < 2) {
    T* dst = static_cast<T*>(kind == 0 ? p.dst[0] : p.dst[1]);
    const int64_t dst_head = kind == 0 ? p.dst_head[0] : p.dst_head[1];
    if (dst) {
      dst += token * (kind == 0 ? p.dst_token[0] : p.dst_token[1]);
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        if (head0 + i >= heads) break;
#pragma unroll
        for (int t = 0; t < ITERS; ++t) {
          if (WHOLE && valid0[t] == 0) continue;
          store_values(dst + (head0 + i) * dst_head + at0[t], WHOLE ? V : valid0[t], a[i][t]);
          store_values(dst + (head0 + i) * dst_head + at1[t], WHOLE ? V : valid1[t], b[i][t]);
        }
      }
    }
  }
  if (kind == 0 || p.held < 0) return;
  const int64_t slot = load_index(p.slots, p.slots64, token * p.slots_stride);
  if (slot < 0 || slot >= (int64_t)p.cache.pages * p.cache.page_size) return;  // a lane's whole group
  const uint32_t page = (uint32_t)slot / (uint32_t)p.cache.page_size;
  const uint32_t offset = (uint32_t)slot - page * (uint32_t)p.cache.page_size;
  const int64_t row = page * p.cache.page + offset * p.cache.token;
  uint8_t* held = kind == 1 ? p.cache.keys : p.cache.values;
  float* scales = kind == 1 ? p.cache.key_scale : p.cache.value_scale;
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    if (head0 + i >= heads) break;
    const int64_t at = row + (head0 + i) * p.cache.head;
#pragma unroll
    for (int t = 0; t < ITERS; ++t)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        a[i][t][v] = rounded<T>(a[i][t][v]);
        b[i][t][v] = rounded<T>(b[i][t][v]);
      }
    float unit = 1.f;
    if (p.held == OMNI_DTYPE_FP8_E4M3) {
      float amax = 0.f;
#pragma unroll
      for (int t = 0; t < ITERS; ++t) {
        float part = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) part = fmaxf(part, fmaxf(fabsf(a[i][t][v]), fabsf(b[i][t][v])));
        amax = fmaxf(amax, WHOLE && valid0[t] == 0 ? 0.f : part);
      }
      for (int off = 1; off < lanes; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
      const float scale = group_scale(amax, &unit);
      if (lane == 0)
        scales[page * p.cache.scale_page + (head0 + i) * p.cache.scale_head +
               offset * p.cache.scale_token] = scale;
    }
#pragma unroll
    for (int t = 0; t < ITERS; ++t) {
      if (WHOLE && valid0[t] == 0) continue;
      if (p.held == OMNI_DTYPE_FP8_E4M3) {
        store_bytes(held + at + at0[t], valid0[t], a[i][t], unit);
        store_bytes(held + at + at1[t], valid1[t], b[i][t], unit);
      } else if (p.held == OMNI_DTYPE_BF16) {
        store_values(reinterpret_cast<__bf16*>(held) + at + at0[t], valid0[t], a[i][t]);
        store_values(reinterpret_cast<__bf16*>(held) + at + at1[t], valid1[t], b[i][t]);
      } else {
        store_values(reinterpret_cast<_Float16*>(held) + at + at0[t], valid0[t], a[i][t]);
        store_values(reinterpret_cast<_Float16*>(held) + at + at1[t], valid1[t], b[i][t]);
      }
    }
  }
}

template <typename T, int V, int ITERS, int HP, bool WHOLE>
int launch_heads(HeadsParams p, int64_t tokens, hipStream_t stream) {
  for (int kind = 0; kind < 3; ++kind) p.groups[kind] = (p.heads[kind] + HP - 1) / HP;
  p.items = tokens * (p.groups[0] + p.groups[1] + p.groups[2]);
  const int64_t workgroups = ((p.items << p.lane_shift) + 255) / 256;
  if (workgroups > kMostWorkgroups) return OMNI_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((heads_kernel<T, V, ITERS, HP, WHOLE>), dim3((unsigned)workgroups), dim3(256), 0, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

// Up to four heads share a lane's sines and cosines once such lanes fill the chip twice over; fewer
// tokens are a chain of loads, and the shorter the more heads there are side by side.
template <typename T, int V, int ITERS>
int launch_chunks(HeadsParams p, int64_t tokens, hipStream_t stream) {
  p.turned_chunks = p.pairs / V;
  p.chunks = p.turned_chunks + (p.dim - 2 * p.pairs + 2 * V - 1) / (2 * V);
  for (p.lane_shift = 0; (1 << p.lane_shift) * ITERS < p.chunks;) ++p.lane_shift;
  const int64_t lanes = (tokens * (p.heads[0] + p.heads[1] + p.heads[2]) / 4) << p.lane_shift;
  const bool many = lanes >= 512 * 256;
  if constexpr (V > 1) {
    if ((p.dim - 2 * p.pairs) % (2 * V) == 0)
      return many ? launch_heads<T, V, ITERS, 4, true>(p, tokens, stream)
                  : launch_heads<T, V, ITERS, 1, true>(p, tokens, stream);
  }
  return many ? launch_heads<T, V, ITERS, 4, false>(p, tokens, stream)
              : launch_heads<T, V, ITERS, 1, false>(p, tokens, stream);
}

// V: the most of 8, 4, 1 that divide the pairs (or, where nothing is turned, half the head); a head of
// up to 512 values is then at most 64 lanes of ITERS chunks.
template <typename T>
int launch_type(const HeadsParams& p, int64_t tokens, hipStream_t stream) {
  const int runs = p.pairs > 0 ? p.pairs : p.dim / 2;
  if (p.dim % 2 == 0 && runs % 8 == 0) return launch_chunks<T, 8, 1>(p, tokens, stream);
  if (p.dim % 2 == 0 && runs % 4 == 0) return launch_chunks<T, 4, 2>(p, tokens, stream);
  return launch_chunks<T, 1, 4>(p, tokens, stream);
}

struct ReadParams {
  CacheView cache;
  const void* slots;
  int slots64;
  int64_t slots_stride;
  void* dst[2];
  int64_t dst_token[2], dst_head[2];
  int64_t items;  // tokens * kv_heads * chunks
  int kv_heads, chunks;
};

// A lane takes 16 values of a key row and of its value row: 16 or 32 bytes of each.
template <typename H, typename T>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= p.items) return;
  const int64_t rest = item / p.chunks;
  const int chunk = (int)(item - rest * p.chunks);
  const int64_t token = rest / p.kv_heads;
  const int head = (int)(rest - token * p.kv_heads);
  const int64_t slot = load_index(p.slots, p.slots64, token * p.slots_stride);
  const bool held = slot >= 0 && slot < (int64_t)p.cache.pages * p.cache.page_size;
  const uint32_t page = held ? (uint32_t)slot / (uint32_t)p.cache.page_size : 0;
  const uint32_t offset = held ? (uint32_t)slot - page * (uint32_t)p.cache.page_size : 0;
  const int64_t at = page * p.cache.page + head * p.cache.head + offset * p.cache.token + chunk * 16;
  float v[2][16];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* rows = i ? p.cache.values : p.cache.keys;
    if constexpr (std::is_same<H, uint8_t>::value) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(rows + at);
      const float scale = (i ? p.cache.value_scale : p.cache.key_scale)[page * p.cache.scale_page +
                                                                        head * p.cache.scale_head +
                                                                        offset * p.cache.scale_token];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i][4 * j] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 0) * scale;
        v[i][4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 1) * scale;
        v[i][4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 2) * scale;
        v[i][4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 3) * scale;
      }
    } else {
      load_values(reinterpret_cast<const H*>(rows) + at, 16, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!held) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[i][j] = 0.f;
    }
    store_values(static_cast<T*>(p.dst[i]) + token * p.dst_token[i] + head * p.dst_head[i] + chunk * 16,
                 16, v[i]);
  }
}

template <typename H, typename T>
int launch_read(const ReadParams& p, hipStream_t stream) {
  const int64_t workgroups = (p.items + 255) / 256;
  if (workgroups > kMostWorkgroups) return OMNI_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((read_kernel<H, T>), dim3((unsigned)workgroups), dim3(256), 0, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

template <typename H>
int launch_read_as(const ReadParams& p, int dtype, hipStream_t stream) {
  switch (dtype) {
    case OMNI_DTYPE_F32: return launch_read<H, float>(p, stream);
    case OMNI_DTYPE_BF16: return launch_read<H, __bf16>(p, stream);
    case OMNI_DTYPE_F16: return launch_read<H, _Float16>(p, stream);
    default: return OMNI_ERR_INVALID_ARG;
  }
}

bool index_type(int dtype) { return dtype == OMNI_DTYPE_I32 || dtype == OMNI_DTYPE_I64; }

}  // namespace

extern "C" int omni_norm_rotary(const omni_norm_rotary_args* a, omni_stream_t stream) {
  if (!a || a->tokens < 0 || a->heads < 0 || a->kv_heads < 0 || a->heads + a->kv_heads < 1 ||
      a->dim < 1 || a->pairs < 0 || 2 * a->pairs > a->dim || a->heads > 65536 || a->kv_heads > 65536)
    return OMNI_ERR_INVALID_ARG;
  if (a->dtype != OMNI_DTYPE_F32 && a->dtype != OMNI_DTYPE_BF16 && a->dtype != OMNI_DTYPE_F16)
    return OMNI_ERR_INVALID_ARG;
  if (a->layout != OMNI_ROTARY_HALF && a->layout != OMNI_ROTARY_INTERLEAVED)
    return OMNI_ERR_INVALID_ARG;
  if (a->dim > 512) return OMNI_ERR_UNSUPPORTED;
  const int size = a->dtype == OMNI_DTYPE_F32 ? 4 : 2;
  HeadsParams p{};
  p.held = -1;
  if (a->cache) {
    if (!index_type(a->slots_dtype) || a->cache->dim != a->dim || a->cache->kv_heads != a->kv_heads ||
        a->kv_heads < 1 || !cache_view(*a->cache, 1, &p.cache))
      return OMNI_ERR_INVALID_ARG;
    const int held_size = a->cache->dtype == OMNI_DTYPE_FP8_E4M3 ? 1 : 2;
    if (!aligned_to(a->cache->keys, held_size) || !aligned_to(a->cache->values, held_size))
      return OMNI_ERR_INVALID_ARG;
    p.held = a->cache->dtype;
  }
  if (a->tokens == 0) return OMNI_OK;
  if (a->heads > 0 && (!a->q || !a->q_out)) return OMNI_ERR_INVALID_ARG;
  if (a->kv_heads > 0 && (!a->k || (!a->k_out && !a->cache))) return OMNI_ERR_INVALID_ARG;
  if (a->cache && (!a->v || !a->slots || !aligned_to(a->slots, a->slots_dtype == OMNI_DTYPE_I64 ? 8 : 4)))
    return OMNI_ERR_INVALID_ARG;
  if (a->pairs > 0 && (!a->positions || !a->inv_freq || !index_type(a->positions_dtype) ||
                       !aligned_to(a->inv_freq, 8) ||
                       !aligned_to(a->positions, a->positions_dtype == OMNI_DTYPE_I64 ? 8 : 4)))
    return OMNI_ERR_INVALID_ARG;
  if (!aligned_to(a->q, size) || !aligned_to(a->k, size) || !aligned_to(a->v, size) ||
      !aligned_to(a->q_out, size) || !aligned_to(a->k_out, size) || !aligned_to(a->q_weight, 4) ||
      !aligned_to(a->k_weight, 4))
    return OMNI_ERR_INVALID_ARG;
  p.src[0] = a->q;
  p.src[1] = a->k;
  p.src[2] = a->v;
  p.src_token[0] = a->q_stride_token;
  p.src_token[1] = a->k_stride_token;
  p.src_token[2] = a->v_stride_token;
  p.src_head[0] = a->q_stride_head;
  p.src_head[1] = a->k_stride_head;
  p.src_head[2] = a->v_stride_head;
  p.dst[0] = a->q_out;
  p.dst[1] = a->k_out;
  p.dst_token[0] = a->q_out_stride_token;
  p.dst_token[1] = a->k_out_stride_token;
  p.dst_head[0] = a->q_out_stride_head;
  p.dst_head[1] = a->k_out_stride_head;
  p.weight[0] = a->q_weight;
  p.weight[1] = a->k_weight;
  p.positions = a->positions;
  p.positions64 = a->positions_dtype == OMNI_DTYPE_I64;
  p.position_stride = a->positions_stride;
  p.inv_freq = a->inv_freq;
  p.factor = a->factor;
  p.eps = a->eps;
  p.normed = a->normed ? 1 : 0;
  p.interleaved = a->layout == OMNI_ROTARY_INTERLEAVED;
  p.slots = a->slots;
  p.slots64 = a->slots_dtype == OMNI_DTYPE_I64;
  p.slots_stride = a->slots_stride;
  p.heads[0] = (int)a->heads;
  p.heads[1] = (int)a->kv_heads;
  p.heads[2] = a->cache ? (int)a->kv_heads : 0;
  p.pairs = (int)a->pairs;
  p.dim = (int)a->dim;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case OMNI_DTYPE_F32: return launch_type<float>(p, a->tokens, s);
    case OMNI_DTYPE_BF16: return launch_type<__bf16>(p, a->tokens, s);
    default: return launch_type<_Float16>(p, a->tokens, s);
  }
}

extern "C" int omni_read_cache(const omni_read_cache_args* a, omni_stream_t stream) {
  ReadParams p{};
  if (!a || !a->cache || a->tokens < 0 || !index_type(a->slots_dtype)) return OMNI_ERR_INVALID_ARG;
  const omni_kv_cache& cache = *a->cache;
  if (cache.kv_heads < 1 || cache.dim < 16 || cache.dim % 16 || cache.kv_heads > 65536 ||
      cache.dim > 65536 || !cache_view(cache, 16, &p.cache))
    return OMNI_ERR_INVALID_ARG;
  if (a->dtype != OMNI_DTYPE_F32 && a->dtype != OMNI_DTYPE_BF16 && a->dtype != OMNI_DTYPE_F16)
    return OMNI_ERR_INVALID_ARG;
  if (a->tokens == 0) return OMNI_OK;
  const int size = a->dtype == OMNI_DTYPE_F32 ? 4 : 2;
  if (!a->slots || !aligned_to(a->slots, a->slots_dtype == OMNI_DTYPE_I64 ? 8 : 4) || !a->k || !a->v ||
      !aligned_to(a->k, size) || !aligned_to(a->v, size))
    return OMNI_ERR_INVALID_ARG;
  p.slots = a->slots;
  p.slots64 = a->slots_dtype == OMNI_DTYPE_I64;
  p.slots_stride = a->slots_stride;
  p.dst[0] = a->k;
  p.dst[1] = a->v;
  p.dst_token[0] = a->k_stride_token;
  p.dst_token[1] = a->v_stride_token;
  p.dst_head[0] = a->k_stride_head;
  p.dst_head[1] = a->v_stride_head;
  p.kv_heads = (int)cache.kv_heads;
  p.chunks = (int)(cache.dim / 16);
  p.items = a->tokens * p.kv_heads * p.chunks;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (cache.dtype) {
    case OMNI_DTYPE_FP8_E4M3: return launch_read_as<uint8_t>(p, a->dtype, s);
    case OMNI_DTYPE_BF16: return launch_read_as<__bf16>(p, a->dtype, s);
    default: return launch_read_as<_Float16>(p, a->dtype, s);
  }
}
