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
// A workgroup takes a tile of a row's vocabulary. The dense part of the work, the mask, streams
// through it and looks at nothing else. The history's tokens that fall into the tile are counted in
// LDS (integer atomics, whose order changes nothing); whoever finds a token's word empty
// puts it on a list, and the listed tokens and bias entries, few beside the tile, are computed one to
// a thread and stored over the dense part's values. (Looking every logit's count up instead took 20 instructions
// a logit: 200 x 50257 in bf16 16.7 us, 64 x 131072 in float32 with everything 25.9.)
//
// HBM would bound it (64 x 131072 in float32 13.7 us); what does is a workgroup's chain, of which a call
// of one round of workgroups hides nothing: lengths, tokens and bias entries, then the logits and mask
// words, then the counts, then the values (23.7 us; the mask alone 12.8, with histories 17.8).
#include <type_traits>

#include "block_fp8.h"

namespace {

constexpr int kThreads = 512;
constexpr int kTile = kThreads * 16;  // logits

// A token's word in LDS: whether it is in the prompt, in the bias list, and how often it was made.
// 16 bits hold the count of any history shorter than 2^14: half the LDS of 32-bit words, and the
// workgroups a CU holds, with them the bytes in flight, end with LDS.
template <bool WIDE>
struct Word {
  static constexpr int kBits = WIDE ? 32 : 16;
  static constexpr uint32_t kSeen = 1u << (kBits - 1), kBiased = 1u << (kBits - 2), kMade = kBiased - 1u;
  static constexpr int kDwords = kTile * kBits / 32;
  OMNI_DEVICE static uint32_t get(const uint32_t* words, uint32_t at) {
    return WIDE ? words[at] : (words[at >> 1] >> (at & 1) * 16) & 0xffffu;
  }
  // adds `how` (1 or a flag) and returns the word as it was
  OMNI_DEVICE static uint32_t update(uint32_t* words, uint32_t at, uint32_t how) {
    uint32_t* word = WIDE ? words + at : words + (at >> 1);
    const int shift = WIDE ? 0 : (at & 1) * 16;
    const uint32_t old = how == 1u ? atomicAdd(word, how << shift) : atomicOr(word, how << shift);
    return WIDE ? old : (old >> shift) & 0xffffu;
  }
};
constexpr int64_t kNarrowHistory = 1 << 14;
constexpr int64_t kMaxHistory = (1 << 30) - 1;  // tokens: kMade of the wide words

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
template <typename L, typename O, typename H, bool WIDE>
__global__ void __launch_bounds__(kThreads, 8) adjust_logits_kernel(const LogitParams p) {
  constexpr int CHUNK = 16 / sizeof(L), CHUNKS = 16 / CHUNK;  // a thread's 16-byte loads
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  uint32_t* counts = lds;
  using W = Word<WIDE>;
  uint32_t* listed_count = lds + W::kDwords;
  uint16_t* list = reinterpret_cast<uint16_t*>(lds + W::kDwords + 4);  // the tile's tokens that have a word
  const int64_t row = blockIdx.x / p.tiles;
  const int64_t v0 = (int64_t)(blockIdx.x - row * p.tiles) * kTile;
  const int tid = threadIdx.x;

  // the row's tokens first: what names them is two dependent loads away
  const H* tokens = nullptr;
  int length = 0, prompt = 0;
  if (p.history) {
    const int64_t slot = p.slot_index ? p.slot_index[row] : row;
    if (slot >= 0 && slot < p.slots) {
      const int64_t held = load_index(p.lengths, p.lengths64, slot);
      const int64_t first = p.prompt_lengths ? load_index(p.prompt_lengths, p.lengths64, slot) : 0;
      length = (int)(held < p.capacity ? held : p.capacity);
      length = held < 0 ? 0 : length;
      prompt = first < 0 ? 0 : (int)(first < length ? first : length);
      tokens = static_cast<const H*>(p.history) + slot * p.history_stride;
    }
  }
  const bool touches = length > 0 || p.biases > 0;  // of the row: uniform
  const int64_t tile_tokens = p.vocab - v0 < kTile ? p.vocab - v0 : kTile;
  const H* biased = static_cast<const H*>(p.bias_tokens) + row * p.bias_tokens_stride;
  const float* bias_values = p.bias_values + row * p.bias_values_stride;
  // 16-byte loads, all of a round's before the first is used; the first round goes out ahead of the
  // logits. It is counted after they have come, though: each mask word below is waited for under its
  // branch, and with it all that went out before.
  constexpr int PER_LOAD = 16 / sizeof(H), LOADS = 2, ROUND = kThreads * PER_LOAD * LOADS;
  H held[LOADS][PER_LOAD];
  auto load_round = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const int at = base + (q * kThreads + tid) * PER_LOAD;
#pragma unroll
      for (int e = 0; e < PER_LOAD; ++e) held[q][e] = (H)-1;
      if (at < length) {
        if (at + PER_LOAD <= p.capacity) {
          __builtin_memcpy(held[q], tokens + at, 16);
        } else {
#pragma unroll
          for (int e = 0; e < PER_LOAD; ++e)
            if (at + e < length) held[q][e] = tokens[at + e];
        }
      }
    }
  };
  if (length > 0) load_round(0);
  // the same for this thread's bias entry
  const bool has_entry = tid < p.biases;
  const H entry_token = has_entry ? biased[tid] : (H)-1;
  const float entry_value = has_entry ? bias_values[tid] : 0.f;
  // and 64 entries of the list in each wave's lanes, ids outside the vocabulary as -1 (looked at, and so
  // waited for, before the logits go out)
  auto load_entries = [&](int64_t base) __attribute__((always_inline)) {
    const int64_t i = base + (tid & 63);
    const int64_t token = i < p.biases ? (int64_t)biased[i] : -1;
    return token >= 0 && token < p.vocab ? (int)token : -1;
  };
  constexpr int EARLY = 2;
  int early[EARLY];
#pragma unroll
  for (int q = 0; q < EARLY; ++q) early[q] = load_entries(q * 64);
  float l[CHUNKS][CHUNK];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int64_t v = v0 + (i * kThreads + tid) * CHUNK;
    load_values(static_cast<const L*>(p.logits) + row * p.logits_stride + v, p.vocab - v, l[i]);
  }
  uint32_t bits[CHUNKS];
  int64_t mask = -1;
  if (p.allowed) mask = p.allowed_index ? p.allowed_index[row] : row;
  const bool masked = mask >= 0 && mask < p.masks;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int64_t v = v0 + (i * kThreads + tid) * CHUNK;
    bits[i] = 0xffu;
    if (masked && v < p.vocab)
      bits[i] = (uint32_t)p.allowed[mask * p.allowed_stride + (v >> 5)] >> (v & 31);
  }

  // Entry i of the bias list speaks for its token if the token is in the tile and no later entry names
  // it. The wave walks the list 64 entries at a time, one in each lane.
  auto speaks = [&](int64_t i, H token, bool there) __attribute__((always_inline)) {
    const int64_t at = (int64_t)token - v0;
    bool last = there && at >= 0 && at < tile_tokens;
    if (__ballot(last) == 0ull) return false;
    auto walk = [&](int64_t base, int narrow) __attribute__((always_inline)) {
      const int before = (int)(i - base);  // bit operations: no branch to an entry
      uint32_t same = 0u;
#pragma unroll 16
      for (int j = 0; j < 64; ++j)
        same |= (uint32_t)(j > before) & (uint32_t)(__builtin_amdgcn_readlane(narrow, j) == (int)token);
      last = last & (same == 0u);
    };
#pragma unroll
    for (int q = 0; q < EARLY; ++q)
      if (q * 64 < p.biases) walk(q * 64, early[q]);
    for (int64_t base = EARLY * 64; base < p.biases; base += 64) walk(base, load_entries(base));
    return last;
  };
  const bool entry_speaks = p.biases > 0 && speaks(tid, entry_token, has_entry);
  uint32_t listed = 0;
  if (touches) {
    for (int i = tid * 4; i < W::kDwords; i += kThreads * 4)
      *reinterpret_cast<u32x4*>(counts + i) = u32x4{0u, 0u, 0u, 0u};
    if (tid == 0) *listed_count = 0u;
    __syncthreads();
    auto add = [&](int64_t token, uint32_t how) __attribute__((always_inline)) {
      const int64_t at = token - v0;
      if (at < 0 || at >= tile_tokens) return;
      if (W::update(counts, (uint32_t)at, how) == 0u && how != W::kBiased) list[atomicAdd(listed_count, 1u)] = (uint16_t)at;
    };
    for (int base = 0; base < length; base += ROUND) {
      if (base > 0) load_round(base);
#pragma unroll
      for (int q = 0; q < LOADS; ++q)
#pragma unroll
        for (int e = 0; e < PER_LOAD; ++e) {
          const int i = base + (q * kThreads + tid) * PER_LOAD + e;
          if (i < length) add((int64_t)held[q][e], i < prompt ? W::kSeen : 1u);
        }
    }
    for (int i = tid; i < p.biases; i += kThreads) add((int64_t)biased[i], W::kBiased);
    __syncthreads();
    listed = *listed_count;
  }

  const float repetition = p.repetition ? p.repetition[row] : 1.f;
  const float frequency = p.frequency ? p.frequency[row] : 0.f;
  const float presence = p.presence ? p.presence[row] : 0.f;
  O* out = static_cast<O*>(p.out) + row * p.out_stride;
  // A named token's value. Where out is the logits themselves, the dense part may have stored over
  // the logit: the same value, or the -infinity that the mask makes of it here too.
  auto named_value = [&](uint32_t at, uint32_t c, float bias) __attribute__((always_inline)) {
    const int64_t v = v0 + at;
    float t = (float)static_cast<const L*>(p.logits)[row * p.logits_stride + v];
    const uint32_t word = masked ? (uint32_t)p.allowed[mask * p.allowed_stride + (v >> 5)] : ~0u;
    if (c & ~W::kBiased) t = t > 0.f ? t / repetition : t * repetition;
    if (const uint32_t made = c & W::kMade) t -= frequency * (float)made + presence;
    if (c & W::kBiased) t += bias;
    return (O)((word >> (v & 31)) & 1u ? t : -__builtin_huge_valf());
  };
  // this thread's listed token (unless a bias entry speaks for it) and bias entry, ahead of the dense
  // part's stores
  uint32_t first_at = 0;
  bool first_mine = false;
  O first = (O)0.f, entry = (O)0.f;
  if (tid < listed) {
    first_at = list[tid];
    const uint32_t c = W::get(counts, first_at);
    first_mine = !(c & W::kBiased);
    if (first_mine) first = named_value(first_at, c, 0.f);
  }
  const uint32_t entry_at = entry_speaks ? (uint32_t)((int64_t)entry_token - v0) : 0u;
  if (entry_speaks) entry = named_value(entry_at, W::get(counts, entry_at), entry_value);

#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int64_t v = v0 + (i * kThreads + tid) * CHUNK;
#pragma unroll
    for (int e = 0; e < CHUNK; ++e)
      l[i][e] = (bits[i] >> e) & 1u ? l[i][e] : -__builtin_huge_valf();
    store_values(out + v, p.vocab - v, l[i]);
  }
  if (!touches) return;
  __syncthreads();  // the dense part's stores are done
  if (first_mine) out[v0 + first_at] = first;
  if (entry_speaks) out[v0 + entry_at] = entry;
  for (uint32_t i = tid + kThreads; i < listed; i += kThreads) {
    const uint32_t at = list[i], c = W::get(counts, at);
    if (!(c & W::kBiased)) out[v0 + at] = named_value(at, c, 0.f);
  }
  for (int64_t i0 = kThreads; i0 < p.biases; i0 += kThreads) {  // of whole waves
    const int64_t i = i0 + tid;
    const H token = i < p.biases ? biased[i] : (H)-1;
    if (!speaks(i, token, i < p.biases)) continue;
    const uint32_t at = (uint32_t)((int64_t)token - v0);
    out[v0 + at] = named_value(at, W::get(counts, at), bias_values[i]);
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
  if (a->history && (!a->lengths || a->capacity < 0 || a->capacity > kMaxHistory ||
                     a->history_stride < a->capacity ||
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
  // a tile's words and, with its length, the list of those in use: no more than tokens and entries
  const int64_t touched = (a->history ? a->capacity : 0) + a->biases;
  const bool wide = a->history && a->capacity >= kNarrowHistory;
  const unsigned lds = touched ? (unsigned)(((wide ? Word<true>::kDwords : Word<false>::kDwords) + 4) * 4 +
                                            2 * (touched < kTile ? touched : kTile))
                               : 0u;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto* l, auto* o) -> int {
    using L = std::remove_pointer_t<decltype(l)>;
    using O = std::remove_pointer_t<decltype(o)>;
    const dim3 grid((unsigned)(a->rows * p.tiles)), block(kThreads);
    auto kernel = a->tokens_dtype == OMNI_DTYPE_I64
                      ? (wide ? adjust_logits_kernel<L, O, int64_t, true> : adjust_logits_kernel<L, O, int64_t, false>)
                      : (wide ? adjust_logits_kernel<L, O, int32_t, true> : adjust_logits_kernel<L, O, int32_t, false>);
    hipLaunchKernelGGL(kernel, grid, block, lds, s, p);
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
