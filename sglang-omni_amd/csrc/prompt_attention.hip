// Attention of whole prompts: packed sequences, each with its own number of queries and keys, heads
// grouped over key heads,
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i . k_j) / sum_j exp(scale q_i . k_j)
//
// over the keys j that query i sees: all of its sequence, or with `causal` those up to its own place
// when the last query stands at the last key. A query that sees none is zero.
//
// One pass over the keys with the running maximum m and sum l of a softmax. A wave owns 32 rows; a row
// is a (query, head) pair, the heads of a group side by side, so that a tile of keys in shared memory
// serves the whole group. Scores are computed transposed, S^T = K Q^T (32 x 32 x 16 MFMAs, a lane's
// column one row's scores), so that a row's maximum is a lane's own but for one swap of half-waves, and
// P^T is the B operand of O^T = V^T P^T as it stands: of each 16 keys, lanes below 32 hold 0 .. 3 and 8
// .. 11, the others 4 .. 7 and 12 .. 15, and V^T, read transposed, takes its keys in that order. The
// weights are rounded to the rows' type for that product (half a step of each, the sum l is of the
// unrounded ones); scores, maxima, sums and outputs are float32.
//
// The matrix cores bound long prompts, and the clock that falls under them: 16384 tokens of 32 heads over 8
// of 128, causal, 1950 - 2010 us, 1094 - 1128 TFLOP/s (a library's 8192^3 product 1237). Per 64 keys a wave
// has 1024 cycles of MFMAs and about 670 of the softmax's, which another wave's MFMAs hide. Short ones are
// latency: 37 tokens 7 us, bounds, then keys and queries, a tile or two, the join.
#include <type_traits>

#include "attention.h"

namespace {

struct PromptParams {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint8_t* out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;  // bytes
  const void* starts;
  const void* key_starts;
  int wide;  // the starts are int64
  int tokens, key_tokens;  // tokens * group below 2^31
  int sequences;
  int cleared;  // the rows in front of the first sequence and behind the last one become zero
  int kv_heads, group, dim, causal;
  float scale;  // of the scores, times log2(e)
  int splits;   // workgroups that share a row tile's keys
  float* parts;  // with several: [splits][tokens][heads][dim], then [splits][tokens][heads][2] of m and l
};

constexpr float kLazy = 6.f;
constexpr int keys_of(int dim, bool long_form) { return long_form && dim < 256 ? 64 : 32; }  // of a tile

OMNI_DEVICE int start_of(const void* starts, int wide, int at, int end) {
  const int64_t s = wide ? static_cast<const int64_t*>(starts)[at]
                         : (int64_t) static_cast<const int32_t*>(starts)[at];
  return (int)(s < 0 ? 0 : s > end ? end : s);
}

// The LDS slot, of 16 bytes, that piece p of key row r takes in its row: K's rows are read 16 bytes a
// lane, 32 consecutive rows the same piece; V's transposed, 8 consecutive rows 4 pieces of each.
template <int D>
OMNI_DEVICE int k_slot(int r, int p) {
  return D == 64 ? p ^ ((r >> 1) & 7) : p ^ (r & 15);
}
template <int D>
OMNI_DEVICE int v_slot(int r, int p) {
  return D == 64 ? p ^ (((r >> 1) & 1) * 4) : p ^ ((r & 3) * 4);
}

// LONG: the waves own 32 rows each and share the tiles, [2][K, V] in shared memory, the next one on its
// way. Not LONG, for few rows: the waves share 32 rows and each owns every NW-th tile, [NW][K, V], and
// their parts are joined at the end; so many more workgroups, each with fewer tiles one after the other.
template <typename T, int D, int NW, bool LONG>
__global__ void __launch_bounds__(64 * NW, D == 64 ? 3 : D == 128 ? 2 : 1) prompt_kernel(const PromptParams p) {
  using O = Op<T>;
  constexpr int kRows = LONG ? 32 * NW : 32;
  constexpr int kKeys = keys_of(D, LONG), kBlocks = kKeys / 32, kSteps = kKeys / 16;
  constexpr int kPieces = D / 8;  // 16-byte pieces of a row
  constexpr int kTile = kKeys * D * 2;
  // DMA instructions a wave and tile; their offsets repeat after 16 rows
  constexpr int kDma = kKeys * kPieces / 64 / (LONG ? NW : 1);
  constexpr int kOffsets = LONG ? kDma : kDma / kSteps;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, half = lane >> 5, column = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

  // Key head fastest: the 8 XCDs take workgroups in turn, so with 8 (4, 2) key heads each XCD's L2
  // holds its own head's keys. The last tiles of a sequence, which see the most keys, go first.
  const int kv_head = blockIdx.x % p.kv_heads;
  const int split = blockIdx.x / p.kv_heads % p.splits;
  const int slot = blockIdx.x / p.kv_heads / p.splits;
  // Sequence s owns the tiles from floor(first row / kRows) + s on: never fewer than it needs, and
  // found by search without a sum over the sequences before it: 64 at a time, each lane one's bounds.
  // Rows that are cleared are two more sequences, the first and the last, without keys.
  int lo = 0, n = p.sequences + 2 * p.cleared;
  int first, last, key_first, key_last;
  for (;;) {
    const int step = (n + 63) / 64, at = lane * step;
    int f = 0, l = 0, kf = 0, kl = 0;
    if (at < n) {
      const int s = lo + at - p.cleared;  // -1: the rows in front, p.sequences: those behind
      f = s < 0 ? 0 : start_of(p.starts, p.wide, s, p.tokens);
      l = s == p.sequences ? p.tokens : start_of(p.starts, p.wide, s + 1, p.tokens);
      if (s >= 0 && s < p.sequences) {
        kf = start_of(p.key_starts, p.wide, s, p.key_tokens);
        kl = start_of(p.key_starts, p.wide, s + 1, p.key_tokens);
      }
    }
    const bool before = at < n && f * p.group / kRows + lo + at <= slot;
    const int count = __builtin_popcountll(__ballot(before)), found = count > 0 ? count - 1 : 0;
    lo += found * step;
    if (step == 1) {
      first = __builtin_amdgcn_readlane(f, found);
      last = __builtin_amdgcn_readlane(l, found);
      key_first = __builtin_amdgcn_readlane(kf, found);
      key_last = __builtin_amdgcn_readlane(kl, found);
      break;
    }
    n = n - found * step < step ? n - found * step : step;
  }
  const int queries = last - first, rows = queries * p.group;
  const int at_slot = slot - (first * p.group / kRows + lo), row_tiles = (rows + kRows - 1) / kRows;
  if (queries <= 0 || at_slot < 0 || at_slot >= row_tiles) return;
  const int row0 = (row_tiles - 1 - at_slot) * kRows;
  const int keys = key_last > key_first ? key_last - key_first : 0;

  // this lane's row, and how many keys it, the wave's first and last row and the tile's last see
  const int wave_row = row0 + (LONG ? wave * 32 : 0);
  const int row = wave_row + column < rows ? wave_row + column : rows - 1;
  const int query = (uint32_t)row / (uint32_t)p.group;
  const int head = kv_head * p.group + row - query * p.group;
  const int ahead = p.causal ? keys - queries + 1 : keys;
  auto seen_by = [&](int r) __attribute__((always_inline)) {
    const int s = p.causal ? (int)((uint32_t)(r < rows ? r : rows - 1) / (uint32_t)p.group) + ahead : ahead;
    return s < 0 ? 0 : s;
  };
  const int seen = seen_by(row);
  const int seen_least = seen_by(wave_row), seen_most = wave_row < rows ? seen_by(wave_row + 31) : 0;
  // this workgroup's tiles of them
  const int all_tiles = (seen_by(row0 + kRows - 1) + kKeys - 1) / kKeys;
  const int share = (all_tiles + p.splits - 1) / p.splits;
  const int low = split * share, high = low + share < all_tiles ? low + share : all_tiles;

  // DMA: instruction i of the wave fills slots 64 i .. of its part of the tile; the row and piece that
  // belong there
  uint32_t k_off[kOffsets], v_off[kOffsets];
#pragma unroll
  for (int i = 0; i < kOffsets; ++i) {
    const int at = ((LONG ? wave * kDma : 0) + i) * 64 + lane, r = at / kPieces, s = at % kPieces;
    const int kp = k_slot<D>(r, s), vp = v_slot<D>(r, s);
    k_off[i] = kp * 8 < p.dim ? (uint32_t)(r * p.k_token + kp * 16) : kOutOfRange;
    v_off[i] = vp * 8 < p.dim ? (uint32_t)(r * p.v_token + vp * 16) : kOutOfRange;
  }
  const uint8_t* k_base = p.k + (int64_t)key_first * p.k_token + kv_head * p.k_head;
  const uint8_t* v_base = p.v + (int64_t)key_first * p.v_token + kv_head * p.v_head;
  // rows behind the sequence's last key are zeros
  auto issue_rows = [&](const uint8_t* base, int64_t pitch, const uint32_t (&off)[kOffsets], int tile,
                        uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < kDma / kOffsets; ++g) {
      const int at = tile * kKeys + g * 16;
      const int valid = keys - at < kKeys ? keys - at : kKeys;
      const u32x4 rsrc =
          dma_rsrc(base + at * pitch, valid > 0 ? (uint32_t)((valid - 1) * pitch + p.dim * 2) : 0u);
#pragma unroll
      for (int i = 0; i < kOffsets; ++i) dma_rows(rsrc, stage + (g * kOffsets + i) * 1024, off[i]);
    }
  };
  const uint32_t place =
      (uint32_t)(uintptr_t)(OMNI_LDS uint8_t*)lds + (LONG ? wave * kDma * 1024 : wave * 2 * kTile);
  auto issue = [&](int tile) __attribute__((always_inline)) {
    const uint32_t stage = place + (LONG ? ((tile - low) & 1) * 2 * kTile : 0);
    issue_rows(k_base, p.k_token, k_off, tile, stage);
    issue_rows(v_base, p.v_token, v_off, tile, stage + kTile);
  };

  const int top_tile = high - 1 - (LONG ? 0 : wave);
  if (top_tile >= low) issue(top_tile);
  typename O::x8 q[D / 16];
  {
    const uint8_t* from = p.q + (int64_t)(first + query) * p.q_token + head * p.q_head + half * 16;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      if (s * 16 + half * 8 < p.dim)
        q[s] = *reinterpret_cast<const typename O::x8*>(from + s * 32);
      else
        q[s] = typename O::x8{};
    }
  }
  // The queries, waited for here with the first tile: in its loop the compiler would wait for them again, and
  // with them for the tile on its way. (Heads of 256 keep them where this would move them from; a chain of
  // the other form is as long either way.)
  if constexpr (LONG && D < 256) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) asm volatile("" : "+v"(q[s]));
  }
  f32x16 o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -__builtin_inff(), m_use = 0.f, l = 0.f;

  // Where this lane reads in a tile: K's row `column` for each step of 16 dimensions (the second 32 keys
  // lie 32 rows on), V's for each block of 32 dimensions (16 keys 16 rows on, an operand's second four 8).
  constexpr int kPitch = D * 2;
  int k_at[D / 16], v_at[D / 32];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) k_at[c] = column * kPitch + k_slot<D>(column, c * 2 + half) * 16;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) {
    const int r = half * 4 + ((lane & 15) >> 2), piece = d * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    v_at[d] = kTile + r * kPitch + v_slot<D>(r, piece) * 16 + (lane & 1) * 8;
  }
  const uint8_t OMNI_LDS* shared = (const uint8_t OMNI_LDS*)lds + (LONG ? 0 : wave * 2 * kTile);
  auto k_operand = [&](int stage, int b, int c) __attribute__((always_inline)) {
    return *(const typename O::x8 OMNI_LDS*)(shared + k_at[c] + (stage * 2 * kTile + b * 32 * kPitch));
  };
  auto v_operand = [&](int stage, int c, int d) __attribute__((always_inline)) {
    const uint8_t OMNI_LDS* at = shared + v_at[d] + (stage * 2 * kTile + c * 16 * kPitch);
    return __builtin_bit_cast(typename O::x8, read_transposed(at, at + 8 * kPitch));
  };
  // the tile has arrived in every wave, and every wave has read the one before, whose place the next
  // one takes
  auto arrive = [&](int tile) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    asm volatile("s_barrier" ::: "memory");
    if (tile > low) issue(tile - 1);
  };
  auto scores_of = [&](int stage, f32x16 (&s)[kBlocks]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) s[b] = O::mfma32(k_operand(stage, b, c), q[c], s[b]);
  };
  // The weights of a tile's scores. The maximum they are taken against moves only where a score is past
  // it by more than 2^kLazy: until then weights are that much larger, which costs no precision, and the
  // sums and outputs need no rescaling.
  auto weights_of = [&](const f32x16 (&s)[kBlocks], typename O::x8 (&w)[kSteps]) __attribute__((always_inline)) {
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = half_max(top) * p.scale;
    if (__ballot(top > m + kLazy) != 0) {
      const float m_new = fmaxf(m, top);
      // a row that has seen nothing yet: its weights are exp2(-infinity - 0)
      m_use = m_new == -__builtin_inff() ? 0.f : m_new;
      const float keep = __builtin_amdgcn_exp2f(m - m_use);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= keep;
    }
    const float shift = O::kBias - m_use;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], p.scale, shift));
        l += x;
        w[b * 2 + i / 8][i % 8] = (T)x;
      }
  };
  auto accumulate = [&](int stage, const typename O::x8 (&w)[kSteps]) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kSteps; ++c)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) o[d] = O::mfma32(v_operand(stage, c, d), w[c], o[d]);
  };

  // 4 dimensions of a row, from d on, out: the result, or where workgroups share the keys a part (without
  // keys that count its maximum and sum alone). Which is which is told by the sum: zero where no score is
  // above -infinity, NaN where one is NaN. The maximum is -infinity also where all are NaN.
  auto store_row = [&](int at_query, int at_head, int d, f32x4 x, float m, float l)
                       __attribute__((always_inline)) {
    const int64_t token = first + at_query;
    if (p.splits > 1) {
      const int64_t heads = (int64_t)p.kv_heads * p.group, at = ((int64_t)split * p.tokens + token) * heads + at_head;
      if (d == 0) {
        float* stats = p.parts + (int64_t)p.splits * p.tokens * heads * p.dim + at * 2;
        stats[0] = m;
        stats[1] = l;
      }
      if (l != 0.f) *reinterpret_cast<f32x4*>(p.parts + at * p.dim + d) = x;
      return;
    }
    const float unit = 1.f / l;
    typename O::x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(l == 0.f ? 0.f : x[e] * unit);
    *reinterpret_cast<typename O::x4*>(p.out + token * p.out_token + at_head * p.out_head + d * 2) = y;
  };
  // The outputs through the matrix cores' pipeline: for code whose paths part and meet right after a product.
  // Where such a meeting is reached straight and by a loop, the compiler counts the wait states before it
  // along the longer way alone, and its copies there read results that are not there yet.
  auto settle = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 3");
    __builtin_amdgcn_sched_barrier(0);
  };
  // what a row does not see: its scores
  auto hide = [&](int first_key, f32x16 (&s)[kBlocks]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = first_key + b * 32 + (i / 4) * 8 + half * 4 + i % 4;
        s[b][i] = key < seen ? s[b][i] : -__builtin_inff();
      }
  };
  // and its values: one that some of these rows do not see may be an infinity or a NaN, and zero times
  // it is one too, so that its keys' sum over zeros is not zero. LONG, whose registers are all in use, looks
  // the tile over at once; else 16 keys at a time, those that only some of the rows see, and those that
  // none sees are passed over (taken so, LONG spills: 24 x 350 tokens of 16 heads 45 -> 52 us).
  auto accumulate_seen = [&](int first_key, int stage, const typename O::x8 (&w)[kSteps])
                             __attribute__((always_inline)) {
    uint32_t bad = 0;
    auto any = [&](const f32x16& zeros) __attribute__((always_inline)) {
      bool some = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) some |= zeros[i] != 0.f;
      return __ballot(some) != 0;
    };
    f32x16 zeros;
    if constexpr (LONG) {
#pragma unroll
      for (int i = 0; i < 16; ++i) zeros[i] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int c = 0; c < kSteps; ++c) zeros = O::mfma32(v_operand(stage, c, d), typename O::x8{}, zeros);
      if (any(zeros)) {
        bad = (1u << kSteps) - 1;
      } else {
        accumulate(stage, w);
        settle();
      }
    } else {
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        const int key = first_key + c * 16;
        if (key >= seen_most) continue;
        typename O::x8 v[D / 32];
#pragma unroll
        for (int d = 0; d < D / 32; ++d) v[d] = v_operand(stage, c, d);
        if (key + 16 > seen_least) {
#pragma unroll
          for (int i = 0; i < 16; ++i) zeros[i] = 0.f;
#pragma unroll
          for (int d = 0; d < D / 32; ++d) zeros = O::mfma32(v[d], typename O::x8{}, zeros);
          if (any(zeros)) {
            bad |= 1u << c;
            continue;
          }
        }
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[d] = O::mfma32(v[d], w[c], o[d]);
        settle();
      }
    }
    if (bad == 0) return;
    // each key's contribution on its own, added where it is seen; rare, so a loop of little code
#pragma unroll 1
    for (int e = 0; e < kKeys; ++e) {
      const int c = e / 16, key = first_key + c * 16 + (e % 8 / 4) * 8 + (e % 16 / 8) * 4 + e % 4;
      if ((bad >> c & 1) == 0) continue;
      const bool mine = half == e % 16 / 8;
      // w[c], by masks: a choice by index would keep w in memory, on every call's way here
      u32x4 bits = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        bits |= __builtin_bit_cast(u32x4, w[i]) & (c == i ? 0xffffffffu : 0u);
      const typename O::x8 wc = __builtin_bit_cast(typename O::x8, bits);
      typename O::x8 we;
#pragma unroll
      for (int j = 0; j < 8; ++j) we[j] = mine && j == e % 8 ? wc[j] : (T)0.f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        const typename O::x8 v = v_operand(stage, c, d);
        typename O::x8 ve;
#pragma unroll
        for (int j = 0; j < 8; ++j) ve[j] = mine && j == e % 8 ? v[j] : (T)0.f;
        f32x16 part;
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] = 0.f;
        part = O::mfma32(ve, we, part);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += key < seen ? part[i] : 0.f;
      }
    }
  };

  if constexpr (LONG) {
    // Tiles from the last: first those that some row of the workgroup does not see whole (and one more
    // where the next would not be in the first stage).
    int tile = high - 1;
    const int whole = seen_by(row0) / kKeys;  // tiles that every row sees
    for (; tile >= low && (tile >= whole || (tile - low) % 2 == 1); --tile) {
      arrive(tile);
      const int first_key = tile * kKeys, stage = (tile - low) & 1;
      if (first_key >= seen_most) continue;
      const bool partial = first_key + kKeys > seen_least;
      f32x16 s[kBlocks];
      typename O::x8 w[kSteps];
      scores_of(stage, s);
      if (partial) hide(first_key, s);
      weights_of(s, w);
      if (partial) {
        accumulate_seen(first_key, stage, w);
      } else {
        accumulate(stage, w);
        settle();
      }
    }
    // then whole tiles, the stage a constant of the code
    auto step = [&](int stage) __attribute__((always_inline)) {
      arrive(tile);
      f32x16 s[kBlocks];
      typename O::x8 w[kSteps];
      scores_of(stage, s);
      weights_of(s, w);
      accumulate(stage, w);
      --tile;
    };
    while (tile > low) {
      step(0);
      step(1);
    }
    if (tile == low) step(0);
  } else {
    int tile = top_tile;
    auto step = [&](auto partial) __attribute__((always_inline)) {
      const int first_key = tile * kKeys;
      f32x16 s[kBlocks];
      typename O::x8 w[kSteps];
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDma) : "memory");  // K is here, V may be on its way
      scores_of(0, s);
      // once K has been read, the next one takes its place, and below so for V
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (tile - NW >= low) issue_rows(k_base, p.k_token, k_off, tile - NW, place);
      if constexpr (partial) hide(first_key, s);
      weights_of(s, w);
      if (tile - NW >= low)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDma) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if constexpr (partial)
        accumulate_seen(first_key, 0, w);
      else
        accumulate(0, w);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (tile - NW >= low) issue_rows(v_base, p.v_token, v_off, tile - NW, place + kTile);
      tile -= NW;
    };
    while (tile >= low && tile * kKeys + kKeys > seen_least) step(std::true_type{});
    while (tile >= low) step(std::false_type{});
    // The waves' parts joined: each leaves its outputs in its own tiles' place, and a thread takes 4
    // dimensions of a row from all of them, in their order.
    constexpr int kLine = D;  // floats
    static_assert(32 * kLine * 4 <= 2 * kTile, "a wave's outputs fit its tiles");
    float* const stats = reinterpret_cast<float*>(lds + NW * 2 * kTile);  // [NW][2][32]
    auto place_of = [](int r, int quad) { return r * kLine + (quad ^ (r & 7)) * 4; };
    l = half_sum(l);
    if (half == 0) {
      stats[wave * 64 + column] = m;
      stats[wave * 64 + 32 + column] = l;
    }
    float* const mine = reinterpret_cast<float*>(lds + wave * 2 * kTile);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(mine + place_of(column, d * 8 + i * 2 + half)) =
            f32x4{o[d][i * 4], o[d][i * 4 + 1], o[d][i * 4 + 2], o[d][i * 4 + 3]};
    __syncthreads();
    for (int item = threadIdx.x; item < 32 * (D / 4); item += 64 * NW) {
      const int r = item / (D / 4), d = item % (D / 4) * 4;
      if (row0 + r >= rows || d >= p.dim) continue;
      float m_all = stats[r];
#pragma unroll
      for (int w = 1; w < NW; ++w) m_all = fmaxf(m_all, stats[w * 64 + r]);
      const float m_base = m_all == -__builtin_inff() ? 0.f : m_all;
      float l_all = 0.f;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float keep = __builtin_amdgcn_exp2f(stats[w * 64 + r] - m_base);
        l_all = __builtin_fmaf(stats[w * 64 + 32 + r], keep, l_all);
        const f32x4 part = *reinterpret_cast<const f32x4*>(lds + w * 2 * kTile + place_of(r, d / 4) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(part[e], keep, x[e]);
      }
      const int at_query = (uint32_t)(row0 + r) / (uint32_t)p.group;
      store_row(at_query, kv_head * p.group + row0 + r - at_query * p.group, d, x, m_all, l_all);
    }
    return;
  }

  l = half_sum(l);
  const bool stored = wave_row + column < rows;
  if (p.splits > 1) {
    if (!stored) return;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d * 32 + i * 8 + half * 4 < p.dim)
          store_row(query, head, d * 32 + i * 8 + half * 4,
                    f32x4{o[d][i * 4], o[d][i * 4 + 1], o[d][i * 4 + 2], o[d][i * 4 + 3]}, m, l);
    return;
  }
  // A lane holds 4 dimensions of each 8; with the other half-wave's of one 8 for its own of the next it
  // stores 16 bytes at a time.
  const bool zero = l == 0.f;
  const float unit = zero ? 0.f : 1.f / l;
  uint8_t* to = p.out + (int64_t)(first + query) * p.out_token + head * p.out_head;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      typename O::x4 x, y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = (T)(o[d][i * 4 + j] * unit);
        y[j] = (T)(o[d][i * 4 + 4 + j] * unit);
      }
      const u32x2 a = __builtin_bit_cast(u32x2, x), b = __builtin_bit_cast(u32x2, y);
      const auto r0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
      const int at = d * 32 + (i + half) * 8;
      const u32x4 all = {r0[0], r1[0], r0[1], r1[1]}, none = {0u, 0u, 0u, 0u};  // none: the values may be NaN
      if (stored && at < p.dim) *reinterpret_cast<u32x4*>(to + at * 2) = zero ? none : all;
    }
}

// The parts of a row's keys joined in their order: 4 dimensions a thread. Rows of no sequence have no
// parts.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const PromptParams p) {
  const int quads = p.dim / 4;
  const int64_t heads = (int64_t)p.kv_heads * p.group, all = p.tokens * heads;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, row = item / quads;
  const int d = (int)(item - row * quads) * 4;
  if (row >= all) return;
  const int token = (int)(row / heads);
  if (!p.cleared && (token < start_of(p.starts, p.wide, 0, p.tokens) ||
                     token >= start_of(p.starts, p.wide, p.sequences, p.tokens)))
    return;
  const float* stats = p.parts + p.splits * all * p.dim;
  float m = -__builtin_inff();
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, stats[(s * all + row) * 2]);
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.splits; ++s) {
    const float sum = stats[(s * all + row) * 2 + 1];
    if (sum == 0.f) continue;  // no part was stored
    const float keep = __builtin_amdgcn_exp2f(stats[(s * all + row) * 2] - m);
    l = __builtin_fmaf(sum, keep, l);
    const f32x4 x = *reinterpret_cast<const f32x4*>(p.parts + (s * all + row) * p.dim + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], keep, o[e]);
  }
  const float unit = l == 0.f ? 0.f : 1.f / l;
  typename Op<T>::x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(o[e] * unit);
  const int head = (int)(row - token * heads);
  *reinterpret_cast<typename Op<T>::x4*>(p.out + token * p.out_token + head * p.out_head + d * 2) = y;
}

template <typename T, int D, int NW, bool LONG>
int launch_prompt(PromptParams p, hipStream_t stream) {
  constexpr int kTiles = 2 * keys_of(D, LONG) * D * 2;
  constexpr int kLds = LONG ? 2 * kTiles : NW * (kTiles + 64 * 4);
  const int64_t slots = (int64_t)p.tokens * p.group / (LONG ? 32 * NW : 32) + p.sequences + 2 * p.cleared;
  const int64_t quads = (int64_t)p.tokens * p.kv_heads * p.group * (p.dim / 4);
  const int64_t joins = p.splits > 1 ? (quads + 255) / 256 : 0;
  if (slots * p.kv_heads * p.splits > kMostWorkgroups || joins > kMostWorkgroups) return OMNI_ERR_UNSUPPORTED;
  if (kLds > 64 * 1024) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(prompt_kernel<T, D, NW, LONG>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess)
      return OMNI_ERR_LAUNCH;
  }
  hipLaunchKernelGGL((prompt_kernel<T, D, NW, LONG>), dim3((unsigned)(slots * p.kv_heads * p.splits)),
                     dim3(64 * NW), kLds, stream, p);
  OMNI_LAUNCH_CHECK();
  if (joins > 0) {
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)joins), dim3(256), 0, stream, p);
    OMNI_LAUNCH_CHECK();
  }
  return OMNI_OK;
}

struct Plan {
  bool long_form;
  int splits;
};

// The form and the number of workgroups that share a row tile's keys: the least of their estimated times
// in us, which come from what the host knows, so with sequences taken to be of one length. Of each form:
// a workgroup's start and end on a CU that others share, its time a step (64 keys of 128 rows, or 128 of
// 32) there, and a step's time in a chain of them. Fitted to 37 .. 8192 tokens of 8 .. 32 heads alone and
// in batches, and 1 .. 1000 tokens after 4000 .. 100000 keys; the choice is the fastest measured one or
// within 20 % of it. 1000 tokens of 16 heads over 8: 15.7 us not LONG, 26.3 LONG; 8192 of them 370 and
// 292; 500 tokens of 32 heads after 20000 keys 218 not LONG, 391 LONG, 175 LONG in four pieces.
Plan plan_of(int64_t tokens, int64_t key_tokens, int64_t sequences, int64_t heads, int64_t kv_heads,
             int64_t dim, bool causal) {
  struct Cost {
    double start, step, chain;
  };
  constexpr Cost kCosts[3][2] = {{{1.8, 0.36, 0.6}, {3.0, 0.52, 0.83}},
                                 {{3.0, 0.72, 0.9}, {4.0, 0.97, 1.1}},
                                 {{6.0, 1.8, 1.8}, {8.0, 3.1, 3.2}}};
  const Cost* costs = kCosts[dim <= 64 ? 0 : dim <= 128 ? 1 : 2];
  const double count = sequences > 0 ? (double)sequences : 1.0;
  const double keys = key_tokens / count, queries = tokens / count;
  const double seen = causal ? (queries < keys ? keys - queries / 2 : keys / 2) : keys;
  const double rows = (double)tokens * (heads / kv_heads);
  Plan best = {false, 1};
  double least = 1e30;
  for (int form = 0; form < 2; ++form) {
    const double tiles = (rows / (form ? 128 : 32) + count) * kv_heads, width = form ? 64 : 128;
    for (int splits = 1; splits <= 32 && (splits == 1 || keys >= 256.0 * splits); splits *= 2) {
      const double busy = tiles * splits / 256;
      const double shared = busy * (costs[form].start + costs[form].step * seen / width / splits);
      const double alone = keys / width / splits * costs[form].chain * (form && busy > 1 ? 1.4 : 1.0);
      const double parts = (double)tokens * heads * (dim + 2) * 8 * splits;  // bytes there and back
      const double joined = splits > 1 ? 6 + 0.4 * splits + parts / 4e6 : 0;
      const double time = (form ? 1.0 : 0.0) + (shared > alone ? shared : alone) + joined;
      if (time < least) {
        least = time;
        best = {form == 1, splits};
      }
    }
  }
  return best;
}

template <typename T>
int launch_dim(const PromptParams& p, bool long_form, hipStream_t stream) {
  if (p.dim <= 64)
    return long_form ? launch_prompt<T, 64, 4, true>(p, stream) : launch_prompt<T, 64, 4, false>(p, stream);
  if (p.dim <= 128)
    return long_form ? launch_prompt<T, 128, 4, true>(p, stream) : launch_prompt<T, 128, 4, false>(p, stream);
  return long_form ? launch_prompt<T, 256, 4, true>(p, stream) : launch_prompt<T, 256, 4, false>(p, stream);
}

}  // namespace

extern "C" int64_t omni_prompt_plan(int64_t tokens, int64_t key_tokens, int64_t sequences, int64_t heads,
                                    int64_t kv_heads, int64_t dim, int causal, int* tile_rows) {
  Plan plan = {false, 1};
  if (tokens > 0 && key_tokens > 0 && heads > 0 && kv_heads > 0 && sequences >= 0)
    plan = plan_of(tokens, key_tokens, sequences, heads, kv_heads, dim, causal != 0);
  if (tile_rows) *tile_rows = plan.long_form ? 128 : 32;
  return plan.splits;
}

extern "C" int omni_prompt_attention(const omni_prompt_args* a, omni_stream_t stream) {
  if (!a || a->tokens < 0 || a->key_tokens < 0 || a->sequences < 0 || a->heads < 1 || a->kv_heads < 1 ||
      a->heads % a->kv_heads || a->heads > 65536 || a->dim < 8 || a->dim % 8 || !(a->scale > 0.f) ||
      !(a->scale <= 1e30f) || a->sequences > 0x7ffffff0LL ||
      (a->dtype != OMNI_DTYPE_BF16 && a->dtype != OMNI_DTYPE_F16) ||
      (a->starts_dtype != OMNI_DTYPE_I32 && a->starts_dtype != OMNI_DTYPE_I64))
    return OMNI_ERR_INVALID_ARG;
  if (a->dim > 256 || a->key_tokens > 0x7fffff00LL || a->tokens > 0x7fffff00LL ||
      a->tokens * (a->heads / a->kv_heads) > 0x7fffff00LL)
    return OMNI_ERR_UNSUPPORTED;
  const int64_t strides[] = {a->q_stride_token, a->q_stride_head, a->k_stride_token, a->k_stride_head,
                             a->v_stride_token, a->v_stride_head, a->out_stride_token, a->out_stride_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return OMNI_ERR_INVALID_ARG;
  // a tile's keys lie within a buffer's 2 GiB
  if (a->k_stride_token > (1 << 23) || a->v_stride_token > (1 << 23)) return OMNI_ERR_UNSUPPORTED;
  const int index = a->starts_dtype == OMNI_DTYPE_I64 ? 8 : 4;
  if (a->tokens == 0 || (a->sequences == 0 && !a->clear_rest)) return OMNI_OK;
  if (!a->q || !a->out || !a->starts || !a->key_starts || (a->key_tokens > 0 && (!a->k || !a->v)) ||
      !aligned_to(a->q, 16) || !aligned_to(a->k, 16) || !aligned_to(a->v, 16) || !aligned_to(a->out, 16) ||
      !aligned_to(a->starts, index) || !aligned_to(a->key_starts, index))
    return OMNI_ERR_INVALID_ARG;
  PromptParams p{};
  p.q = static_cast<const uint8_t*>(a->q);
  p.k = static_cast<const uint8_t*>(a->k);
  p.v = static_cast<const uint8_t*>(a->v);
  p.out = static_cast<uint8_t*>(a->out);
  p.q_token = a->q_stride_token * 2;
  p.q_head = a->q_stride_head * 2;
  p.k_token = a->k_stride_token * 2;
  p.k_head = a->k_stride_head * 2;
  p.v_token = a->v_stride_token * 2;
  p.v_head = a->v_stride_head * 2;
  p.out_token = a->out_stride_token * 2;
  p.out_head = a->out_stride_head * 2;
  p.starts = a->starts;
  p.key_starts = a->key_starts;
  p.wide = a->starts_dtype == OMNI_DTYPE_I64;
  p.tokens = (int)a->tokens;
  p.key_tokens = (int)a->key_tokens;
  p.cleared = a->clear_rest ? 1 : 0;
  p.sequences = (int)a->sequences;
  p.kv_heads = (int)a->kv_heads;
  p.group = (int)(a->heads / a->kv_heads);
  p.dim = (int)a->dim;
  p.causal = a->causal ? 1 : 0;
  p.scale = a->scale * kLog2e;
  int tile_rows;
  p.splits = (int)omni_prompt_plan(a->tokens, a->key_tokens, a->sequences, a->heads, a->kv_heads, a->dim,
                                   a->causal, &tile_rows);
  p.parts = static_cast<float*>(a->workspace);
  if (p.splits > 1 && (!a->workspace || !aligned_to(a->workspace, 16) ||
                       a->workspace_bytes < p.splits * a->tokens * a->heads * (a->dim + 2) * 4))
    return OMNI_ERR_INVALID_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return a->dtype == OMNI_DTYPE_BF16 ? launch_dim<__bf16>(p, tile_rows == 128, s)
                                     : launch_dim<_Float16>(p, tile_rows == 128, s);
}
