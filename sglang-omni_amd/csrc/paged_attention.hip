// Attention of one new token of each sequence over its paged key-value cache:
//
//   o = sum_j p_j v_j,   p_j = exp(scale q . k_j) / sum_j exp(scale q . k_j),   j < length
//
// for every head, the heads of a group over one key head. Rows of E4M3 count scale_j times their bytes.
// A sequence without keys is zero. Keys on a page outside the cache are left out.
//
// The cache is read once, and that bounds it: 2 x 131072 keys of 8 heads of 128 in 100 us in 8 bits (5.5
// TB/s; a plain read of 1 GiB 6.3, a copy 5.06) and 187 in bf16 (5.7), 64 streams up to 5000 in 139 - 143
// (5.1 - 5.3); one stream of 300 in 7.6, a chain of loads: length, table, rows. (In a graph, as below.) A
// sequence's keys are cut into chunks whose size follows from its length alone, so that a row's bits do not
// depend on the batch; a workgroup takes a chunk of a key head for up to 16 query heads, its four waves every
// fourth tile of 32 keys each, with their own running maximum and sum, joined through shared memory. One
// chunk is the result; several are joined by a second launch, in their order.
//
// Scores transposed, S^T = K Q^T (16 x 16 x 32 MFMAs, K's rows from memory straight into operands: the
// dimensions of a row in any order, so long as q's are in the same), and O^T = V^T P^T as in the prompt
// kernel, V read transposed from shared memory. bf16 weights are held as a sum of two bf16 numbers, 16
// bits of each weight: the matrix cores have nothing else to do here. float16 ones are one number: 11 bits,
// as many as the result is rounded to (9 streams up to 20000: 2.3e-4 from float64 in the mean square, the
// rounding alone 2.0e-4). 8-bit rows widen exactly; the keys' scales multiply the scores and the values'
// the weights.
#include <initializer_list>
#include <type_traits>

#include "attention.h"

namespace {

struct PagedParams {
  const uint8_t* q;
  uint8_t* out;
  int64_t q_row, q_head, out_row, out_head;  // bytes
  CacheView cache;
  const int32_t* table;
  int64_t table_row;
  const void* lengths;
  int wide;
  int64_t columns;  // of the table
  int batch, kv_heads, group, head_tiles, dim;
  float scale;  // of the scores, times log2(e)
  float* parts;  // [batch][heads][chunks][dim], then [batch][heads][chunks][2] of maximum and sum
  int chunks;    // most that a sequence has
  int64_t max_length;
};

constexpr int kKeys = 32;  // of a tile
constexpr int kWaves = 4;
constexpr float kLazy = 6.f;
constexpr int kLeastChunk = 256, kMostChunk = 1024;

// The keys of a chunk, by a sequence's length and the workgroups that share its chunks (a key head's 16
// query heads each). Short chunks spread one stream over the chip, long ones have fewer starts and parts:
// with 256, 512 and 1024 for all lengths and 8 key heads 1 x 2000 takes 10.4, 12.3 and 17.1 us, 1 x 9000 14.1,
// 14.3 and 19.7, 64 up to 5000 157, 147 and 140, 2 x 131072 127, 116 and 103 (E4M3); over 2 key heads 9 up to
// 20000 15.5, 16.3 and 18.4: fewer heads leave more of the chip to the chunks. Up to 512 keys are one chunk,
// which needs no second launch.
__host__ __device__ inline int units_of(int kv_heads, int head_tiles) {
  return kv_heads * head_tiles < 8 ? kv_heads * head_tiles : 8;
}
__host__ __device__ inline int chunk_of(int64_t length, int units) {
  return length <= 2 * kLeastChunk            ? 2 * kLeastChunk
         : length * units <= 64 * kLeastChunk ? kLeastChunk
         : length * units <= 512 * kLeastChunk ? 2 * kLeastChunk
                                              : kMostChunk;
}

// The keys that sequence b's query sees: within the table's room and max_length.
OMNI_DEVICE int length_of(const PagedParams& p, int b) {
  const int64_t given = p.wide ? static_cast<const int64_t*>(p.lengths)[b]
                               : (int64_t) static_cast<const int32_t*>(p.lengths)[b];
  const int64_t room = p.columns * p.cache.page_size, most = room < p.max_length ? room : p.max_length;
  return (int)(given < 0 ? 0 : given > most ? most : given);
}

// Eight E4M3 bytes as bf16 or float16, exactly.
template <typename T>
OMNI_DEVICE typename Op<T>::x8 widen(uint32_t lo, uint32_t hi);
template <>
OMNI_DEVICE bf16x8 widen<__bf16>(uint32_t lo, uint32_t hi) {
  return widen8((int)lo, (int)hi);
}
template <>
OMNI_DEVICE f16x8 widen<_Float16>(uint32_t lo, uint32_t hi) {
  const i32x4 w = {
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.f, false)),
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.f, true)),
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.f, false)),
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.f, true))};
  return __builtin_bit_cast(f16x8, w);
}

// The largest (the sum) over the four lanes that hold a query's scores: lanes 16 and 32 apart.
OMNI_DEVICE float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
OMNI_DEVICE float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// V's LDS slot, of 16 bytes, of piece p of row r: read transposed, 4 rows 2 pieces of each at a time.
template <int D>
OMNI_DEVICE int v_slot(int r, int p) {
  return D == 64 ? p ^ (((r >> 1) & 3) * 2) : p ^ ((r & 7) * 2);
}

// T: the type of q and out, H: of the cache's rows (uint8_t: E4M3). 16-bit rows are T. Weights go into the
// product as PT: bf16 where the values' scales multiply them, whose range float16 has not.
template <typename T, typename H, int D>
__global__ void __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) paged_kernel(const PagedParams p) {
  constexpr bool kBytes = std::is_same<H, uint8_t>::value;
  using PT = typename std::conditional<kBytes, __bf16, T>::type;
  using O = Op<T>;
  using P = Op<PT>;
  constexpr bool kTwo = std::is_same<PT, __bf16>::value;
  constexpr int kPieces = D / 8;  // 16-byte pieces of a row of values in shared memory
  constexpr int kRow = D * (int)sizeof(H);
  constexpr int kLoads = kRow / 64;        // 16-byte loads a lane and 16 keys: 4 lanes to a row
  constexpr int kVLoads = kKeys * kRow / 1024;
  // keys' rows (element offsets, negative: left out), their scales, V tiles of the waves; at the end
  // the waves' outputs
  __shared__ int64_t rows[kMostChunk];
  __shared__ __attribute__((aligned(16))) float scales[kBytes ? 2 : 1][kBytes ? kMostChunk : 4];
  __shared__ __attribute__((aligned(16))) uint8_t tiles[kWaves][kKeys * D * 2];
  __shared__ float stats[kWaves][2][16];

  const int lane = threadIdx.x & 63, column = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int chunk = blockIdx.x;
  const int kv_head = blockIdx.y / p.head_tiles, head_tile = blockIdx.y % p.head_tiles;
  const int b = blockIdx.z;
  const int length = length_of(p, b);
  const int size = chunk_of(length, units_of(p.kv_heads, p.head_tiles));
  const int chunks = (length + size - 1) / size;
  if (chunk > 0 && chunk >= chunks) return;
  const int first = chunk * size, count = length - first < size ? length - first : size;

  // the rows of whole tiles: one past the chunk is left out, as on a page outside the cache
  for (int i = threadIdx.x; i < (count + kKeys - 1) / kKeys * kKeys; i += 64 * kWaves) {
    const uint32_t key = (uint32_t)(first + i), column_of = key / (uint32_t)p.cache.page_size;
    const int page = i < count ? p.table[b * p.table_row + column_of] : -1;
    const uint32_t offset = key - column_of * (uint32_t)p.cache.page_size;
    const bool held = page >= 0 && page < p.cache.pages;
    rows[i] = held ? page * p.cache.page + offset * p.cache.token + kv_head * p.cache.head : -1;
    if constexpr (kBytes) {
      const int64_t at = (int64_t)page * p.cache.scale_page + offset * p.cache.scale_token +
                         kv_head * p.cache.scale_head;
      scales[0][i] = held ? p.cache.key_scale[at] * p.scale : 0.f;
      scales[1][i] = held ? p.cache.value_scale[at] : 0.f;
    }
  }

  // q's operand: lane (column, quarter) holds of head `column` the dimensions that the same lane of a
  // load holds of a key
  const int head_in_group = head_tile * 16 + column;
  const int head = kv_head * p.group + (head_in_group < p.group ? head_in_group : p.group - 1);
  typename O::x8 q[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    // of 16-bit rows load s holds dimensions 32 s + 8 quarter ..; of bytes load s / 2 64 (s / 2) + 16
    // quarter .., its second half for odd s
    const int d = kBytes ? (s / 2) * 64 + quarter * 16 + (s % 2) * 8 : s * 32 + quarter * 8;
    if (d < p.dim)
      q[s] = *reinterpret_cast<const typename O::x8*>(p.q + b * p.q_row + head * p.q_head + d * 2);
    else
      q[s] = typename O::x8{};
  }

  f32x4 o[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), m_use = 0.f, l = 0.f;
  __syncthreads();

  // A tile's rows in registers: loads without branches, so that all are on their way at once. Rows that are
  // left out read the cache's first one.
  u32x4 k[2][kLoads], v[kVLoads];
  const int64_t spare = kv_head * p.cache.head;
  const u32x4 nothing = {0u, 0u, 0u, 0u};
  bool k_whole;  // no row of this lane is left out
  auto load_keys = [&](int at) __attribute__((always_inline)) {
    k_whole = true;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = rows[at + t * 16 + column];
      k_whole &= row >= 0;
      const uint8_t* from = p.cache.keys + (row >= 0 ? row : spare) * sizeof(H);
#pragma unroll
      for (int s = 0; s < kLoads; ++s) {
        const int byte = s * 64 + quarter * 16;
        k[t][s] = *reinterpret_cast<const u32x4*>(from + (byte < p.dim * (int)sizeof(H) ? byte : 0));
      }
    }
  };
  // The values past the caches: nothing reads them again. (A line of keys is read in two halves.) When it was
  // done 2 x 131072 in 8 bits went from 127 to 108 us, 128 x 1000 from 115 to 93; with the keys so too 122 and 110.
  auto load_values_of = [&](int at) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < kVLoads; ++s) {
      const int piece = s * 64 + lane, byte = piece % (kRow / 16) * 16;
      const int64_t row = rows[at + piece / (kRow / 16)];
      v[s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(
          p.cache.values + (row >= 0 ? row : spare) * sizeof(H) +
          (byte < p.dim * (int)sizeof(H) ? byte : 0)));
    }
  };
  uint8_t* const tile = tiles[wave];
  int at = wave * kKeys;
  if (at < count) {
    load_keys(at);
    load_values_of(at);
  }
  for (; at < count; at += kWaves * kKeys) {
    const bool whole = __ballot(!k_whole) == 0;  // the same rows for keys and values
    const int next = at + kWaves * kKeys;
    if (p.dim < D) {  // q is zero behind the head, and so must be what it meets
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int s = 0; s < kLoads; ++s)
          if (s * 64 + quarter * 16 >= p.dim * (int)sizeof(H)) k[t][s] = nothing;
    }
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        typename O::x8 a;
        if constexpr (kBytes)
          a = widen<T>(k[t][c / 2][c % 2 * 2], k[t][c / 2][c % 2 * 2 + 1]);
        else
          a = __builtin_bit_cast(typename O::x8, k[t][c]);
        s[t] = O::mfma16(a, q[c], s[t]);
      }
    }
    if (next < count) load_keys(next);
    if (!whole) {  // what a row left out holds must not meet a weight of zero
#pragma unroll
      for (int i = 0; i < kVLoads; ++i)
        if (rows[at + (i * 64 + lane) / (kRow / 16)] < 0) v[i] = nothing;
    }
    // V to shared memory as it will be read
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int piece = i * 64 + lane, r = piece / (kRow / 16), at16 = piece % (kRow / 16);
      if constexpr (kBytes) {
        const typename P::x8 x = widen<PT>(v[i][0], v[i][1]), y = widen<PT>(v[i][2], v[i][3]);
        *reinterpret_cast<typename P::x8*>(tile + (r * kPieces + v_slot<D>(r, at16 * 2)) * 16) = x;
        *reinterpret_cast<typename P::x8*>(tile + (r * kPieces + v_slot<D>(r, at16 * 2 + 1)) * 16) = y;
      } else {
        *reinterpret_cast<u32x4*>(tile + (r * kPieces + v_slot<D>(r, at16)) * 16) = v[i];
      }
    }
    if (next < count) load_values_of(next);

    // lane (column, quarter) holds keys 16 t + 4 quarter .. + 3 of head `column`
    f32x4 value_scale[2];
    float top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int i = at + t * 16 + quarter * 4;
      if constexpr (kBytes) {
        s[t] *= *reinterpret_cast<const f32x4*>(&scales[0][i]);
        value_scale[t] = *reinterpret_cast<const f32x4*>(&scales[1][i]);
      } else {
        s[t] *= p.scale;
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = rows[i + e] >= 0 ? s[t][e] : -__builtin_inff();
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[t][e]);
    }
    // the maximum moves only where a score is past it by more than 2^kLazy, as in the prompt kernel
    if (__ballot(top > m + kLazy) != 0) {
      const float m_new = fmaxf(m, column_max(top));
      m_use = m_new == -__builtin_inff() ? 0.f : m_new;
      const float keep = __builtin_amdgcn_exp2f(m - m_use);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[d] *= keep;
    }
    const float shift = P::kBias - m_use;
    typename P::x8 w, w_low;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = __builtin_amdgcn_exp2f(s[t][e] + shift);
        l += x;
        if constexpr (kBytes) x *= value_scale[t][e];
        w[t * 4 + e] = (PT)x;
        w_low[t * 4 + e] = (PT)(x - (float)w[t * 4 + e]);
      }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const int r = quarter * 4 + (column >> 2), piece = d * 2 + ((column & 3) >> 1);
      const int within = (column & 1) * 8;
      const typename P::x8 a = __builtin_bit_cast(
          typename P::x8,
          read_transposed((const uint8_t OMNI_LDS*)(tile + (r * kPieces + v_slot<D>(r, piece)) * 16 + within),
                          (const uint8_t OMNI_LDS*)(tile + ((r + 16) * kPieces + v_slot<D>(r + 16, piece)) * 16 +
                                                    within)));
      o[d] = P::mfma16(a, w, o[d]);
      if constexpr (kTwo) o[d] = P::mfma16(a, w_low, o[d]);
    }
  }

  // The waves' parts joined: each leaves its heads' outputs in its tile's place, and a thread takes 4
  // dimensions of a head from all of them, in their order.
  l = column_sum(l);
  if (quarter == 0) {
    stats[wave][0][column] = m;
    stats[wave][1][column] = l;
  }
  static_assert(sizeof(tiles[0]) >= 16 * D * 4, "a wave's outputs fit its tile");
  auto place_of = [](int h, int quad) { return h * D + (quad ^ (h & 15)) * 4; };
  const int heads_here = p.group - head_tile * 16 < 16 ? p.group - head_tile * 16 : 16;
  if (column < heads_here) {
    float* mine = reinterpret_cast<float*>(tile);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(mine + place_of(column, d * 4 + quarter)) = o[d];
  }
  __syncthreads();
  for (int item = threadIdx.x; item < heads_here * (D / 4); item += 64 * kWaves) {
    const int h = item / (D / 4), quad = item % (D / 4), d = quad * 4;
    if (d >= p.dim) continue;
    float m_all = stats[0][0][h];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m_all = fmaxf(m_all, stats[w][0][h]);
    const float m_base = m_all == -__builtin_inff() ? 0.f : m_all;
    float l_all = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float keep = __builtin_amdgcn_exp2f(stats[w][0][h] - m_base);
      l_all = __builtin_fmaf(stats[w][1][h], keep, l_all);
      x += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(tiles[w]) + place_of(h, quad)) * keep;
    }
    const int out_head = kv_head * p.group + head_tile * 16 + h;
    if (chunks > 1) {
      const int64_t at = ((int64_t)b * p.kv_heads * p.group + out_head) * p.chunks + chunk;
      *reinterpret_cast<f32x4*>(p.parts + at * p.dim + d) = x;
      if (quad == 0) {
        float* to = p.parts + (int64_t)p.batch * p.kv_heads * p.group * p.chunks * p.dim + at * 2;
        to[0] = m_all;
        to[1] = l_all;
      }
    } else {
      // Zero by the sum, not by the maximum: that is -infinity where all scores are NaN, too.
      const float unit = 1.f / l_all;
      typename O::x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(l_all == 0.f ? 0.f : x[e] * unit);
      *reinterpret_cast<typename O::x4*>(p.out + b * p.out_row + out_head * p.out_head + d * 2) = y;
    }
  }
}

// The chunks of a (sequence, head) joined: a workgroup of 4 waves, a quarter-wave to a row of up to 64
// dimensions (4 a lane), so 16 chunks at a time, their sums joined in a fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const PagedParams p) {
  constexpr int kQuads = D / 64;  // a lane's, 64 dimensions apart
  const int heads = p.kv_heads * p.group;
  const int b = blockIdx.x / heads, head = blockIdx.x % heads;
  const int length = length_of(p, b);
  const int size = chunk_of(length, units_of(p.kv_heads, p.head_tiles));
  const int chunks = (length + size - 1) / size;
  if (chunks <= 1) return;
  const int64_t at = ((int64_t)b * heads + head) * p.chunks;
  const float* stats = p.parts + (int64_t)p.batch * heads * p.chunks * p.dim + at * 2;
  __shared__ float sums[16][D / 4 + 1][4];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 4, quad = threadIdx.x & 15;
  float m = -__builtin_inff();
  for (int c = lane; c < chunks; c += 64) m = fmaxf(m, stats[2 * c]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
  const float m_use = m == -__builtin_inff() ? 0.f : m;
  float l = 0.f;
  f32x4 o[kQuads];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A quarter-wave's chunks, where there are several up to four at a time, so that their loads are on their way
  // together; one past the last is the last one again, and counts nothing.
  auto add = [&](auto ahead) __attribute__((always_inline)) {
    constexpr int kAhead = decltype(ahead)::value;
    for (int first = part; first < chunks; first += 16 * kAhead) {
      float keep[kAhead], sum[kAhead];
      f32x4 x[kAhead][kQuads];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int c = first + j * 16 < chunks ? first + j * 16 : chunks - 1;
        keep[j] = stats[2 * c];
        sum[j] = stats[2 * c + 1];
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
          if (i * 64 + quad * 4 < p.dim)
            x[j][i] = *reinterpret_cast<const f32x4*>(p.parts + (at + c) * p.dim + i * 64 + quad * 4);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (first + j * 16 >= chunks) break;
        const float weight = __builtin_amdgcn_exp2f(keep[j] - m_use);
        l = __builtin_fmaf(sum[j], weight, l);
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
          if (i * 64 + quad * 4 < p.dim) o[i] += x[j][i] * weight;
      }
    }
  };
  if (chunks > 16)
    add(std::integral_constant<int, D == 256 ? 2 : 4>{});
  else
    add(std::integral_constant<int, 1>{});
#pragma unroll
  for (int i = 0; i < kQuads; ++i) *reinterpret_cast<f32x4*>(sums[part][i * 16 + quad]) = o[i];
  if (quad == 0) sums[part][D / 4][0] = l;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= p.dim) return;
  float total = 0.f, l_all = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    total += sums[i][d / 4][d % 4];
    l_all += sums[i][D / 4][0];
  }
  reinterpret_cast<T*>(p.out + b * p.out_row + head * p.out_head)[d] =
      (T)(l_all == 0.f ? 0.f : total / l_all);
}

template <typename T, typename H, int D>
int launch_paged(const PagedParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((paged_kernel<T, H, D>),
                     dim3((unsigned)p.chunks, (unsigned)(p.kv_heads * p.head_tiles), (unsigned)p.batch),
                     dim3(64 * kWaves), 0, stream, p);
  OMNI_LAUNCH_CHECK();
  if (p.chunks > 1) {
    hipLaunchKernelGGL((join_kernel<T, D>), dim3((unsigned)(p.batch * p.kv_heads * p.group)), dim3(256), 0,
                       stream, p);
    OMNI_LAUNCH_CHECK();
  }
  return OMNI_OK;
}

template <typename T, typename H>
int launch_dim(const PagedParams& p, hipStream_t stream) {
  if (p.dim <= 64) return launch_paged<T, H, 64>(p, stream);
  if (p.dim <= 128) return launch_paged<T, H, 128>(p, stream);
  return launch_paged<T, H, 256>(p, stream);
}

// The most chunks of a length up to `bound`: those of the last length of each chunk size.
int64_t most_chunks(int64_t bound, int kv_heads, int head_tiles) {
  const int units = units_of(kv_heads, head_tiles);
  int64_t most = 1;
  for (int64_t last : {(int64_t)64 * kLeastChunk / units, (int64_t)512 * kLeastChunk / units, bound}) {
    const int64_t length = last < bound ? last : bound, size = chunk_of(length, units);
    const int64_t chunks = (length + size - 1) / size;
    most = chunks > most ? chunks : most;
  }
  return most;
}

}  // namespace

extern "C" int64_t omni_paged_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                                        int64_t max_length) {
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65535 || dim < 1) return 0;
  const int64_t chunks = most_chunks(max_length, (int)kv_heads, (int)((heads / kv_heads + 15) / 16));
  return chunks > 1 ? batch * heads * chunks * (dim + 2) * 4 : 0;
}

extern "C" int omni_paged_attention(const omni_paged_args* a, omni_stream_t stream) {
  if (!a || !a->cache || a->batch < 0 || a->heads < 1 || a->cache->kv_heads < 1 ||
      a->heads % a->cache->kv_heads || a->heads > 65535 || a->cache->dim < 16 || a->cache->dim % 16 ||
      a->table_columns < 0 || a->max_length < 0 || !(a->scale > 0.f) || !(a->scale <= 1e30f) ||
      (a->dtype != OMNI_DTYPE_BF16 && a->dtype != OMNI_DTYPE_F16) ||
      (a->cache->dtype != OMNI_DTYPE_FP8_E4M3 && a->cache->dtype != a->dtype) ||
      (a->lengths_dtype != OMNI_DTYPE_I32 && a->lengths_dtype != OMNI_DTYPE_I64))
    return OMNI_ERR_INVALID_ARG;
  const int64_t strides[] = {a->q_stride_row, a->q_stride_head, a->out_stride_row, a->out_stride_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return OMNI_ERR_INVALID_ARG;
  PagedParams p{};
  if (!cache_view(*a->cache, 16, &p.cache)) return OMNI_ERR_INVALID_ARG;
  if (a->cache->dim > 256 || a->batch > 65535 || a->max_length > 0x7ffffc00LL) return OMNI_ERR_UNSUPPORTED;
  if (a->batch == 0) return OMNI_OK;
  if (!a->q || !a->out || !a->lengths || (a->table_columns > 0 && !a->table) || !aligned_to(a->q, 16) ||
      !aligned_to(a->out, 16) || !aligned_to(a->table, 4) ||
      !aligned_to(a->lengths, a->lengths_dtype == OMNI_DTYPE_I64 ? 8 : 4))
    return OMNI_ERR_INVALID_ARG;
  const int64_t kv_heads = a->cache->kv_heads, group = a->heads / kv_heads;
  const int64_t tiles = (group + 15) / 16;
  if (kv_heads * tiles > 65535) return OMNI_ERR_UNSUPPORTED;
  const int64_t chunks = most_chunks(a->max_length, (int)kv_heads, (int)tiles);
  if (chunks > 1 && a->batch * a->heads > kMostWorkgroups) return OMNI_ERR_UNSUPPORTED;
  if (chunks > 1 && (!a->workspace || !aligned_to(a->workspace, 16) ||
                     a->workspace_bytes < a->batch * a->heads * chunks * (a->cache->dim + 2) * 4))
    return OMNI_ERR_INVALID_ARG;
  p.q = static_cast<const uint8_t*>(a->q);
  p.out = static_cast<uint8_t*>(a->out);
  p.q_row = a->q_stride_row * 2;
  p.q_head = a->q_stride_head * 2;
  p.out_row = a->out_stride_row * 2;
  p.out_head = a->out_stride_head * 2;
  p.table = static_cast<const int32_t*>(a->table);
  p.table_row = a->table_stride;
  p.lengths = a->lengths;
  p.wide = a->lengths_dtype == OMNI_DTYPE_I64;
  p.columns = a->table_columns;
  p.batch = (int)a->batch;
  p.kv_heads = (int)kv_heads;
  p.group = (int)group;
  p.head_tiles = (int)tiles;
  p.dim = (int)a->cache->dim;
  p.scale = a->scale * kLog2e;
  p.parts = static_cast<float*>(a->workspace);
  p.chunks = (int)chunks;
  p.max_length = a->max_length;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool bytes = a->cache->dtype == OMNI_DTYPE_FP8_E4M3;
  if (a->dtype == OMNI_DTYPE_BF16)
    return bytes ? launch_dim<__bf16, uint8_t>(p, s) : launch_dim<__bf16, __bf16>(p, s);
  return bytes ? launch_dim<_Float16, uint8_t>(p, s) : launch_dim<_Float16, _Float16>(p, s);
}
