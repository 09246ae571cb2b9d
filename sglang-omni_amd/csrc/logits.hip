// What a sampler does to a row of logits before it draws from it, in one pass:
//
//   l = logits[b][v]
//   v in the row's history:            l = l > 0 ? l / repetition : l * repetition
//   count(v) of the tokens it made:    l -= frequency * count + presence * (count > 0)
//   v in the row's bias list:          l += bias          (listed twice: the last entry stands)
//   v not allowed by the row's bitmask: l = -infinity
//
// A row's history is a row of a token pool (its slot's, or its own), the first prompt_length tokens
// of which count as seen but not as made. Ids outside the vocabulary are passed over.
//
// A workgroup takes a tile of a row's vocabulary: it counts the history's tokens that fall into the
// tile in LDS (integer atomics, whose order changes nothing) and then streams the tile's logits.
#include <type_traits>

#include "block_fp8.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 2;  // chunks of 8 logits
constexpr int kTile = kThreads * kPerThread * 8;

struct LogitParams {
  const void* logits;
  int64_t logits_stride;
  void* out;
  int64_t out_stride;
  int64_t vocab;
  int tiles;
  const void* history;
  int64_t history_stride, capacity, slots;
  const void* lengths;
  const void* prompt_lengths;
  int lengths64;
  const int64_t* slot_index;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const void* bias_tokens;
  const float* bias_values;
  int64_t bias_tokens_stride, bias_values_stride, biases;
  const int32_t* allowed;
  int64_t allowed_stride, masks;
  const int64_t* allowed_index;
};

OMNI_DEVICE int64_t load_index(const void* p, int wide, int64_t at) {
  return wide ? static_cast<const int64_t*>(p)[at] : (int64_t)static_cast<const int32_t*>(p)[at];
}

// L the logits' type, O the output's, H the history's and bias lists' token type.
template <typename L, typename O, typename H>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(const LogitParams p) {
  extern __shared__ uint32_t lds[];
  uint32_t* counts = lds;                              // bit 31: seen; the rest: times made
  uint32_t* entries = lds + (p.history ? kTile : 0);   // last bias entry + 1 of a token
  const int64_t row = blockIdx.x / p.tiles;
  const int64_t v0 = (int64_t)(blockIdx.x - row * p.tiles) * kTile;
  const int tid = threadIdx.x;

  float l[kPerThread][8];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int64_t v = v0 + (i * kThreads + tid) * 8;
    load_values(static_cast<const L*>(p.logits) + row * p.logits_stride + v, p.vocab - v, l[i]);
  }
  uint32_t bits[kPerThread];
  int64_t mask = -1;
  if (p.allowed) mask = p.allowed_index ? p.allowed_index[row] : row;
  const bool masked = mask >= 0 && mask < p.masks;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int64_t v = v0 + (i * kThreads + tid) * 8;
    bits[i] = 0xffu;
    if (masked && v < p.vocab)
      bits[i] = (uint32_t)p.allowed[mask * p.allowed_stride + (v >> 5)] >> (v & 31);
  }

  const int words = (p.history ? kTile : 0) + (p.biases ? kTile : 0);
  for (int i = tid * 4; i < words; i += kThreads * 4)
    *reinterpret_cast<u32x4*>(lds + i) = u32x4{0u, 0u, 0u, 0u};
  __syncthreads();
  if (p.history) {
    const int64_t slot = p.slot_index ? p.slot_index[row] : row;
    if (slot >= 0 && slot < p.slots) {
      int64_t length = load_index(p.lengths, p.lengths64, slot);
      length = length < p.capacity ? length : p.capacity;
      const int64_t prompt = p.prompt_lengths ? load_index(p.prompt_lengths, p.lengths64, slot) : 0;
      const H* tokens = static_cast<const H*>(p.history) + slot * p.history_stride;
      for (int64_t i = tid; i < length; i += kThreads) {
        const int64_t at = (int64_t)tokens[i] - v0;
        if (at < 0 || at >= kTile || at + v0 >= p.vocab) continue;
        if (i < prompt)
          atomicOr(&counts[at], 0x80000000u);
        else
          atomicAdd(&counts[at], 1u);
      }
    }
  }
  for (int64_t i = tid; i < p.biases; i += kThreads) {
    const int64_t at = (int64_t)static_cast<const H*>(p.bias_tokens)[row * p.bias_tokens_stride + i] - v0;
    if (at >= 0 && at < kTile) atomicMax(&entries[at], (uint32_t)i + 1u);
  }
  __syncthreads();

  const float repetition = p.repetition ? p.repetition[row] : 1.f;
  const float frequency = p.frequency ? p.frequency[row] : 0.f;
  const float presence = p.presence ? p.presence[row] : 0.f;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int at = (i * kThreads + tid) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float t = l[i][e];
      const uint32_t c = p.history ? counts[at + e] : 0u;
      if (c) {
        t = t > 0.f ? t / repetition : t * repetition;
        const uint32_t made = c & 0x7fffffffu;
        if (made) t -= frequency * (float)made + presence;
      }
      if (p.biases) {
        const uint32_t entry = entries[at + e];
        if (entry) t += p.bias_values[row * p.bias_values_stride + entry - 1];
      }
      l[i][e] = (bits[i] >> e) & 1u ? t : -__builtin_huge_valf();
    }
    const int64_t v = v0 + at;
    store_values(static_cast<O*>(p.out) + row * p.out_stride + v, p.vocab - v, l[i]);
  }
}

}  // namespace

extern "C" int omni_adjust_logits(const omni_logits_args* a, omni_stream_t stream) {
  if (!a || a->rows < 0 || a->vocab < 1 || a->vocab > 0x40000000LL) return OMNI_ERR_INVALID_ARG;
  if (a->rows == 0) return OMNI_OK;
  auto size = [](int d) { return d == OMNI_DTYPE_F32 ? 4 : 2; };
  const bool floats = a->dtype == OMNI_DTYPE_F32 || a->dtype == OMNI_DTYPE_BF16 ||
                      a->dtype == OMNI_DTYPE_F16;
  if (!floats || (a->out_dtype != a->dtype && a->out_dtype != OMNI_DTYPE_F32) ||
      (a->tokens_dtype != OMNI_DTYPE_I32 && a->tokens_dtype != OMNI_DTYPE_I64) ||
      (a->lengths_dtype != OMNI_DTYPE_I32 && a->lengths_dtype != OMNI_DTYPE_I64))
    return OMNI_ERR_INVALID_ARG;
  if (!a->logits || !a->out || a->logits_stride < a->vocab || a->out_stride < a->vocab ||
      !aligned_to(a->logits, size(a->dtype)) || !aligned_to(a->out, size(a->out_dtype)))
    return OMNI_ERR_INVALID_ARG;
  const int token_size = a->tokens_dtype == OMNI_DTYPE_I64 ? 8 : 4;
  if (a->history && (!a->lengths || a->capacity < 0 || a->history_stride < a->capacity ||
                     a->slots < 1 || (!a->slot_index && a->slots < a->rows) ||
                     !aligned_to(a->history, token_size)))
    return OMNI_ERR_INVALID_ARG;
  if (a->biases < 0 || (a->biases && (!a->bias_tokens || !a->bias_values ||
                                      a->bias_tokens_stride < 0 || a->bias_values_stride < 0 ||
                                      a->biases > 0x7fffffffLL ||
                                      !aligned_to(a->bias_tokens, token_size))))
    return OMNI_ERR_INVALID_ARG;
  if (a->allowed && (a->allowed_stride < (a->vocab + 31) / 32 || a->masks < 1 ||
                     (!a->allowed_index && a->masks < a->rows) || !aligned_to(a->allowed, 4)))
    return OMNI_ERR_INVALID_ARG;
  LogitParams p{};
  p.logits = a->logits;
  p.logits_stride = a->logits_stride;
  p.out = a->out;
  p.out_stride = a->out_stride;
  p.vocab = a->vocab;
  p.tiles = (int)((a->vocab + kTile - 1) / kTile);
  p.history = a->history;
  p.history_stride = a->history_stride;
  p.capacity = a->capacity;
  p.slots = a->slots;
  p.lengths = a->lengths;
  p.prompt_lengths = a->prompt_lengths;
  p.lengths64 = a->lengths_dtype == OMNI_DTYPE_I64;
  p.slot_index = a->slot_index;
  p.repetition = a->repetition;
  p.frequency = a->frequency;
  p.presence = a->presence;
  p.bias_tokens = a->bias_tokens;
  p.bias_values = a->bias_values;
  p.bias_tokens_stride = a->bias_tokens_stride;
  p.bias_values_stride = a->bias_values_stride;
  p.biases = a->biases;
  p.allowed = a->allowed;
  p.allowed_stride = a->allowed_stride;
  p.masks = a->masks;
  p.allowed_index = a->allowed_index;
  if (a->rows * p.tiles > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  const unsigned lds = ((a->history ? kTile : 0) + (a->biases ? kTile : 0)) * 4;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto* l, auto* o) -> int {
    using L = std::remove_pointer_t<decltype(l)>;
    using O = std::remove_pointer_t<decltype(o)>;
    const dim3 grid((unsigned)(a->rows * p.tiles)), block(kThreads);
    if (a->tokens_dtype == OMNI_DTYPE_I64)
      hipLaunchKernelGGL((adjust_logits_kernel<L, O, int64_t>), grid, block, lds, s, p);
    else
      hipLaunchKernelGGL((adjust_logits_kernel<L, O, int32_t>), grid, block, lds, s, p);
    OMNI_LAUNCH_CHECK();
    return OMNI_OK;
  };
  float* f = nullptr;
  __bf16* b = nullptr;
  _Float16* h = nullptr;
  if (a->dtype == OMNI_DTYPE_F32) return go(f, f);
  if (a->dtype == OMNI_DTYPE_BF16) return a->out_dtype == OMNI_DTYPE_F32 ? go(b, f) : go(b, b);
  return a->out_dtype == OMNI_DTYPE_F32 ? go(h, f) : go(h, h);
}
