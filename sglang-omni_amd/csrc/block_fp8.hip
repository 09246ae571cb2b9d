// Linear layers in 8-bit floating point (OCP E4M3) with a float32 scale for each block of 128:
//
//   y[m][n] = sum_b sx[m][b] * sw[n / 128][b] * (sum_{k in block b} x[m][k] * w[n][k]) (+ bias[n])
//
// block b holds k = 128 b .. 128 b + 127 (the last one shorter), and omni_block_quantize, which
// makes such rows from bf16 / f16 / float32 ones.
//
// Three kernels: few rows (up to 16: the weight's bytes bound it), a ring of LDS stages (tiles up to
// 64 x 128: latency bounds it) and large tiles (128 x 128, 256 x 256: the matrix cores and the
// operand traffic bound it); choose_tile at the end picks by an estimate of each one's time.
#include <type_traits>

#include "block_fp8.h"

namespace {

struct GemmParams {
  const uint8_t* x;
  int64_t x_stride;  // bytes
  const float* xs;
  int64_t xs_row, xs_block;
  const uint8_t* w;
  int64_t w_stride;
  const float* ws;
  int64_t ws_row;  // scales from one block of 128 columns to the next
  int64_t rows, n;
  int k, blocks;
  int x_features;  // float x: the features that are there (k is rounded up to 16)
  const float* bias;
  void* out;
  int64_t out_stride;
  int out_dtype;
  int row_tiles, col_tiles;
  int chunk;  // few rows: K blocks whose products are in LDS at a time
};

// Four consecutive columns of one row, rounded once to the output's type.
template <bool EXACT>
OMNI_DEVICE void store_columns(const GemmParams& p, int64_t row, int64_t col, f32x4 v,
                               const float (&bias)[4]) {
  if (row >= p.rows || col >= p.n) return;
  const float o[4] = {v[0] + bias[0], v[1] + bias[1], v[2] + bias[2], v[3] + bias[3]};
  const int64_t at = row * p.out_stride + col;
  if (!EXACT)
    store_values<__bf16, 4>(static_cast<__bf16*>(p.out) + at, p.n - col, o);
  else if (p.out_dtype == OMNI_DTYPE_F32)
    store_values<float, 4>(static_cast<float*>(p.out) + at, p.n - col, o);
  else
    store_values<_Float16, 4>(static_cast<_Float16*>(p.out) + at, p.n - col, o);
}

// A wave's tiles to its part of the output, through a piece of LDS of its own: 16-byte stores of
// whole runs of a row, where the lanes' own four columns would write every cache line in four parts.
template <typename O, int TM, int TN, int BYTES>
OMNI_DEVICE void store_tile(const GemmParams& p, int64_t row0, int64_t col0, int lane,
                            const f32x4 (&acc)[TM][TN], uint8_t* piece) {
  constexpr int PER_LANE = 16 / sizeof(O);         // values of a 16-byte store
  constexpr int LANES = TN * 16 / PER_LANE;        // lanes of a row
  constexpr int PITCH = TN * 16 * sizeof(O) + 16;  // bytes; the pad spreads a column over the banks
  constexpr int FIT = BYTES / 16 * 16 / (16 * PITCH);
  constexpr int TILES = FIT >= TM ? TM : FIT >= TM / 2 ? TM / 2 : FIT >= 2 ? 2 : 1;  // rows at once
  static_assert(FIT >= 1 && TM % TILES == 0 && LANES <= 64, "epilogue piece");
  const int lr = lane & 15, lq = lane >> 4;
  const int orow = lane / LANES, ocol = lane % LANES * PER_LANE;
  const int64_t col = col0 + ocol, valid = p.n - col;
#pragma unroll
  for (int i0 = 0; i0 < TM; i0 += TILES) {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const f32x4 v = acc[i0 + i][j];
        const float f[4] = {v[0], v[1], v[2], v[3]};
        store_values<O, 4>(reinterpret_cast<O*>(piece + (i * 16 + lr) * PITCH) + j * 16 + lq * 4, 4, f);
      }
#pragma unroll
    for (int r = 0; r < TILES * 16; r += 64 / LANES) {
      const int64_t row = row0 + i0 * 16 + r + orow;
      const u32x4 v = *reinterpret_cast<const u32x4*>(piece + (r + orow) * PITCH + ocol * sizeof(O));
      O* dst = static_cast<O*>(p.out) + row * p.out_stride + col;
      if (row < p.rows) {
        if (valid >= PER_LANE) {
          __builtin_memcpy(dst, &v, 16);
        } else {
          const O* o = reinterpret_cast<const O*>(&v);
#pragma unroll
          for (int e = 0; e < PER_LANE; ++e)
            if (e < valid) dst[e] = o[e];
        }
      }
    }
  }
}

constexpr int kBand = 8;

template <int TN>
OMNI_DEVICE void add_scaled(f32x4 (&acc)[TN], const f32x4 (&part)[TN], float s) {
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = __builtin_fmaf(part[j][e], s, acc[j][e]);
  // the sums are wanted here: moved behind the loop's later MFMAs, they would keep a block's products
  // alive and spill
#pragma unroll
  for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[j]));
}

// A tile of the output by WM x WN waves, each TM x TN MFMA tiles of 16 x 16. A K block's product
// starts from zero, and one fma per element adds it, scaled, to the float32 accumulator.
//
// Rows of 128 bytes travel to LDS by DMA into two buffers, with the rows' scales of the block behind
// them; a row's 16-byte slot s is stored at s ^ (row % 8), so that the operand reads of 16
// rows spread over all banks. A lane's 32 bytes of a row are slots q and q + 4 (q = lane / 16) for
// both operands, so the products of a block pair up whatever order the instruction numbers them in.
//
// Within a block the fmas of one row of tiles stand between the MFMAs of the next. Two barriers a
// block, before the last row of tiles of each half of x: what has been read (w's rows, kept in
// registers, and the first half; the second half) is overwritten from there on by block kt + 2, so
// every DMA has one and a half blocks to arrive, and the MFMAs of that row cover the operand reads
// that follow the barrier.
template <int WM, int WN, int TM, int TN>
struct BlockTile {
  static constexpr int NW = WM * WN;
  static constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
  // 64-lane DMA instructions of a wave: of each half of x's rows, and of w's
  static constexpr int A_HALF = BM / 16 / NW, B_PER_WAVE = BN / 8 / NW;
  static constexpr int SCALE_PARTS = (BM + 63) / 64;  // DMA instructions of 64 scales
  static constexpr int PER_WAVE = 2 * A_HALF + B_PER_WAVE + 1;
  static constexpr int SCALES = SCALE_PARTS * 256;    // bytes, at a stage's start
  static constexpr int STAGE = SCALES + (BM + BN) * kBlock;
  static constexpr int LDS = 2 * STAGE;
  // A block's DMA instructions go out a few per row of tiles: the first FREED (w, scales, x's first
  // half) over rows TM / 2 - 1 .. TM - 2, the rest over row TM - 1 and the next block's rows
  // 0 .. TM / 2 - 2. sent(i): how many have gone out before row i, of the block they belong to.
  static constexpr int FREED = B_PER_WAVE + 1 + A_HALF;
  static constexpr int HALF = TM / 2;
  static constexpr int sent(int i) {
    return i < HALF - 1 ? FREED + A_HALF * (i + 1) / HALF
                        : FREED * (i - HALF + 1) / HALF;
  }
  static constexpr int sent_after(int i) {
    return i < HALF - 1 ? FREED + A_HALF * (i + 2) / HALF
           : i < TM - 1 ? FREED * (i - HALF + 2) / HALF
                        : FREED + A_HALF / HALF;
  }
  static_assert(BM / 16 % NW == 0 && BN / 8 % NW == 0 && TN * 16 <= 128 && TM % 2 == 0, "tile split");
};

template <int WM, int WN, int TM, int TN, bool EXACT>
__global__ void __launch_bounds__(64 * WM * WN, 2) block_fp8_gemm_kernel(const GemmParams p) {
  using T = BlockTile<WM, WN, TM, TN>;
  constexpr int BM = T::BM, BN = T::BN;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int tile = xcd_tile(blockIdx.x, p.row_tiles * p.col_tiles);
  // bands of kBand row tiles, their columns one after the other: the 32 workgroups that an XCD runs
  // at once then share 8 tiles of rows and 4 of columns in its L2, instead of 32 and 1
  const int band = tile / (kBand * p.col_tiles);
  const int band_rows = p.row_tiles - band * kBand < kBand ? p.row_tiles - band * kBand : kBand;
  const int in_band = tile - band * kBand * p.col_tiles;
  const int ct = in_band / band_rows;
  const int64_t m0 = (int64_t)(band * kBand + in_band - ct * band_rows) * BM;
  const int64_t n0 = (int64_t)ct * BN;

  // resources of the tile's own rows: rows past the last read zeros
  const int m_rows = (int)(p.rows - m0 < BM ? p.rows - m0 : BM);
  const int n_rows = (int)(p.n - n0 < BN ? p.n - n0 : BN);
  const auto xr = buffer_rsrc(p.x + m0 * p.x_stride, (uint32_t)((m_rows - 1) * p.x_stride + p.k));
  const auto wr = buffer_rsrc(p.w + n0 * p.w_stride, (uint32_t)((n_rows - 1) * p.w_stride + p.k));
  const auto sr = buffer_rsrc(p.xs + m0 * p.xs_row, (uint32_t)((m_rows - 1) * p.xs_row + (p.blocks - 1) * p.xs_block + 1) * 4u);
  const int drow = lane >> 3;
  const int dslot = ((lane & 7) ^ drow) * 16;  // the byte of the row this lane's DMA piece holds
  // x's rows in two halves, of each wave row the first TM / 2 tiles and the others
  auto a_row = [&](int half, int i) {
    const int g = wave * T::A_HALF + i;
    return g / TM * (TM * 16) + half * (TM * 8) + g % TM * 8;
  };
  uint32_t a_off[2][T::A_HALF], b_off[T::B_PER_WAVE];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < T::A_HALF; ++i) {
      const int row = a_row(h, i) + drow;
      a_off[h][i] = row < m_rows ? (uint32_t)(row * (int)p.x_stride + dslot) : kOutOfRange;
    }
#pragma unroll
  for (int i = 0; i < T::B_PER_WAVE; ++i) {
    const int row = (wave * T::B_PER_WAVE + i) * 8 + drow;
    b_off[i] = row < n_rows ? (uint32_t)(row * (int)p.w_stride + dslot) : kOutOfRange;
  }
  // every wave brings one part of the scales (several the same one, where there are fewer parts)
  const int s_part = wave % T::SCALE_PARTS;
  const int s_row = s_part * 64 + lane;
  const uint32_t s_off = s_row < m_rows ? (uint32_t)(s_row * (int)p.xs_row) * 4u : kOutOfRange;
  const int s_step = (int)p.xs_block * 4;
  // DMA instruction c of block kt: w's pieces and the scales, x's first half, x's second half. The
  // last block may end early, and blocks past it are empty: their pieces read zeros.
  auto issue = [&](int kt, int c) __attribute__((always_inline)) {
    uint8_t* st = lds + (kt & 1) * T::STAGE;
    const bool in = dslot < p.k - kt * kBlock;
    if (c < T::B_PER_WAVE) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr,
          (__attribute__((address_space(3))) void*)(st + T::SCALES + BM * kBlock +
                                                    (wave * T::B_PER_WAVE + c) * 1024),
          16, (int)(in ? b_off[c] : kOutOfRange), kt * kBlock, 0, 0);
    } else if (c == T::B_PER_WAVE) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          sr, (__attribute__((address_space(3))) void*)(st + s_part * 256), 4,
          (int)(kt < p.blocks ? s_off : kOutOfRange), min(kt, p.blocks - 1) * s_step, 0, 0);
    } else {
      const int a = c - T::B_PER_WAVE - 1, half = a / T::A_HALF, piece = a % T::A_HALF;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (__attribute__((address_space(3))) void*)(st + T::SCALES + a_row(half, piece) * kBlock),
          16, (int)(in ? a_off[half][piece] : kOutOfRange), kt * kBlock, 0, 0);
    }
  };

  const int lr = lane & 15, lq = lane >> 4;
  const int rd0 = lr * kBlock + ((lq ^ (lr & 7)) * 16);
  const int rd1 = lr * kBlock + (((lq + 4) ^ (lr & 7)) * 16);
  const int a_base = T::SCALES + wm * TM * 16 * kBlock;
  const int b_base = T::SCALES + (BM + wn * TN * 16) * kBlock;
  const int s_base = (wm * TM * 16 + lr) * 4;

  // the scales of the wave's columns, which lie in one block of 128: 64 K blocks in a register
  const int64_t wcol = n0 + wn * TN * 16;
  const float* ws = p.ws + (wcol < p.n ? wcol / kBlock : 0) * p.ws_row;
  float w_scales = lane < p.blocks ? ws[lane] : 0.f;

  f32x4 acc[TM][TN], part[2][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < TN; ++j) part[(TM - 1) & 1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float s_last = 0.f;

#pragma unroll
  for (int c = 0; c < T::PER_WAVE; ++c) issue(0, c);
#pragma unroll
  for (int c = 0; c < (T::HALF > 1 ? T::sent(0) : T::PER_WAVE); ++c) issue(1, c);
  // A wave's DMAs complete in their order. What a barrier hands over is complete once only the
  // instructions after it, one whole block's, are outstanding in every wave; and with its own LDS
  // reads done too, a wave leaves what it has read to be overwritten.
  auto hand_over = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(T::PER_WAVE) : "memory");
    asm volatile("s_barrier" ::: "memory");
  };
  asm volatile("" : "+v"(w_scales));  // waited for here, and not at every use in the loop
  hand_over();
  i32x8 bytes[TN], av;  // w's operands of the block and x's next one, read one row of tiles ahead
#pragma unroll
  for (int j = 0; j < TN; ++j) bytes[j] = read_operand(lds + b_base + j * 16 * kBlock, rd0, rd1);
  av = read_operand(lds + a_base, rd0, rd1);
  for (int kt = 0, k64 = 64; kt < p.blocks; ++kt) {
    if (kt == k64) {
      w_scales = kt + lane < p.blocks ? ws[kt + lane] : 0.f;
      asm volatile("" : "+v"(w_scales));
      k64 += 64;
    }
    const float sw = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w_scales), kt & 63));
    const uint8_t* st = lds + (kt & 1) * T::STAGE;
    const uint8_t* next = lds + ((kt + 1) & 1) * T::STAGE;
    Operand<EXACT> bv[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) bv[j] = Operand<EXACT>(bytes[j]);
    float s[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) s[i] = *reinterpret_cast<const float*>(st + s_base + i * 64);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const Operand<EXACT> a(av);
      // w and the first half of x read, the second half there; or all of x read, w and the first
      // half of the next block there
      if (i + 1 == TM / 2 || i + 1 == TM) hand_over();
      // block kt + 2's DMAs into what was read, a few per row of tiles: all at once behind the
      // barrier, they would hold up the MFMAs behind them in every wave
#pragma unroll
      for (int c = T::sent(i); c < T::sent_after(i); ++c) issue(kt + (i + 1 < TM / 2 ? 1 : 2), c);
      av = i + 1 < TM ? read_operand(st + a_base + (i + 1) * 16 * kBlock, rd0, rd1)
                      : read_operand(next + a_base, rd0, rd1);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        part[i & 1][j] = block_product(bv[j], a);
        if (i + 1 == TM) bytes[j] = read_operand(next + b_base + j * 16 * kBlock, rd0, rd1);
      }
      // the row of tiles before this one (at i = 0 the last of the block before)
      if (i == 0) {
        add_scaled<TN>(acc[TM - 1], part[1], s_last);
#pragma unroll
        for (int r = 0; r < TM; ++r) s[r] *= sw;
      } else {
        add_scaled<TN>(acc[i - 1], part[(i & 1) ^ 1], s[i - 1]);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x8, EXACT ? 4 : 1, 0);  // MFMAs of a tile
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);              // the fmas of another
        if (i + 1 == TM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    s_last = s[TM - 1];
  }
  add_scaled<TN>(acc[TM - 1], part[(TM - 1) & 1], s_last);

  // lane: row lane % 16 of row tile i, columns 4 (lane / 16) .. + 3 of column tile j
  const int64_t col0 = wcol + lq * 4;
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      float b[4];
      load_values(p.bias + col0 + j * 16, p.n - col0 - j * 16, b);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] += b[e];
    }
  }
  // the stages' LDS is free once every wave's last (empty) DMAs and reads are done
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  asm volatile("s_barrier" ::: "memory");
  uint8_t* piece = lds + wave * (T::LDS / T::NW / 16 * 16);
  const int64_t wrow = m0 + wm * TM * 16;
  if (!EXACT)
    store_tile<__bf16, TM, TN, T::LDS / T::NW>(p, wrow, wcol, lane, acc, piece);
  else if (p.out_dtype == OMNI_DTYPE_F32)
    store_tile<float, TM, TN, T::LDS / T::NW>(p, wrow, wcol, lane, acc, piece);
  else
    store_tile<_Float16, TM, TN, T::LDS / T::NW>(p, wrow, wcol, lane, acc, piece);
}

template <int WM, int WN, int TM, int TN, bool EXACT>
int launch_gemm(GemmParams p, hipStream_t stream) {
  using T = BlockTile<WM, WN, TM, TN>;
  constexpr int BM = T::BM, BN = T::BN, lds_bytes = T::LDS;
  if (BM * p.x_stride >= (int64_t)kOutOfRange || BN * p.w_stride >= (int64_t)kOutOfRange)
    return OMNI_ERR_UNSUPPORTED;
  const int64_t rt = (p.rows + BM - 1) / BM, ct = (p.n + BN - 1) / BN;
  if (rt * ct > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  p.row_tiles = (int)rt;
  p.col_tiles = (int)ct;
  auto k = block_fp8_gemm_kernel<WM, WN, TM, TN, EXACT>;
  static const bool raised = hipFuncSetAttribute((const void*)k,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 lds_bytes) == hipSuccess;
  if (!raised) return OMNI_ERR_LAUNCH;
  hipLaunchKernelGGL(k, dim3((unsigned)(rt * ct)), dim3(64 * WM * WN), lds_bytes, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

// ------------------------------------------------------------------------------ ring of stages
//
// Tiles that leave a workgroup a CU of its own, or nearly: there the chain of barriers and LDS round
// trips is the time, not the matrix cores. So G blocks to a stage, S stages in a ring, one barrier a
// stage, and every stage but the one in use in flight. 64 x 4096 -> 4096 on 32 x 32 tiles: 9.5 us, 1.85
// TB/s (two buffers and a barrier per block 16 - 19; K split over a workgroup's waves 16).
template <int WM, int WN, int TM, int TN, int S, int G>
struct RingTile {
  static constexpr int NW = WM * WN;
  static constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
  static constexpr int A_PER_WAVE = G * BM / 8 / NW, B_PER_WAVE = G * BN / 8 / NW;
  static constexpr int SCALE_PARTS = (G * BM + 63) / 64;  // DMA instructions of 64 scales
  static constexpr int S_PER_WAVE = (SCALE_PARTS + NW - 1) / NW;
  static constexpr int PER_WAVE = A_PER_WAVE + B_PER_WAVE + S_PER_WAVE;
  static constexpr int SCALES = SCALE_PARTS * 256;
  static constexpr int BLOCK = (BM + BN) * kBlock;
  static constexpr int STAGE = SCALES + G * BLOCK;
  static constexpr int LDS = S * STAGE;
  static_assert(G * BM / 8 % NW == 0 && G * BN / 8 % NW == 0 && TN * 16 <= 128 && 64 % G == 0, "split");
  static_assert((S - 1) * PER_WAVE <= 63 && LDS <= 160 * 1024, "ring");
};

template <int WM, int WN, int TM, int TN, int S, int G, bool EXACT>
__global__ void __launch_bounds__(64 * WM * WN) block_fp8_ring_kernel(const GemmParams p) {
  using T = RingTile<WM, WN, TM, TN, S, G>;
  constexpr int BM = T::BM, BN = T::BN;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  // row tiles inner, each XCD a contiguous range: its workgroups share w's columns in its L2
  const int tile = xcd_tile(blockIdx.x, p.row_tiles * p.col_tiles);
  const int ct = tile / p.row_tiles;
  const int64_t m0 = (int64_t)(tile - ct * p.row_tiles) * BM;
  const int64_t n0 = (int64_t)ct * BN;
  const int m_rows = (int)(p.rows - m0 < BM ? p.rows - m0 : BM);
  const int n_rows = (int)(p.n - n0 < BN ? p.n - n0 : BN);
  const auto xr = buffer_rsrc(p.x + m0 * p.x_stride, (uint32_t)((m_rows - 1) * p.x_stride + p.k));
  const auto wr = buffer_rsrc(p.w + n0 * p.w_stride, (uint32_t)((n_rows - 1) * p.w_stride + p.k));
  const auto sr = buffer_rsrc(p.xs + m0 * p.xs_row, (uint32_t)((m_rows - 1) * p.xs_row + (p.blocks - 1) * p.xs_block + 1) * 4u);
  const int drow = lane >> 3;
  const int dslot = ((lane & 7) ^ drow) * 16;
  uint32_t a_off[T::A_PER_WAVE], b_off[T::B_PER_WAVE], s_off[T::S_PER_WAVE];
  int s_block[T::S_PER_WAVE];
#pragma unroll
  for (int i = 0; i < T::A_PER_WAVE; ++i) {
    const int c = wave * T::A_PER_WAVE + i, row = c % (BM / 8) * 8 + drow;
    a_off[i] = row < m_rows ? (uint32_t)(row * (int)p.x_stride + dslot) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < T::B_PER_WAVE; ++i) {
    const int c = wave * T::B_PER_WAVE + i, row = c % (BN / 8) * 8 + drow;
    b_off[i] = row < n_rows ? (uint32_t)(row * (int)p.w_stride + dslot) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < T::S_PER_WAVE; ++i) {
    const int at = (wave * T::S_PER_WAVE + i) % T::SCALE_PARTS * 64 + lane, row = at % BM;
    s_block[i] = at / BM;
    s_off[i] = row < m_rows && s_block[i] < G
                   ? (uint32_t)(row * (int)p.xs_row + s_block[i] * (int)p.xs_block) * 4u
                   : kOutOfRange;
  }
  // the pieces past the end of K (of its last block, or of whole blocks) read zeros
  auto issue = [&](int stage) __attribute__((always_inline)) {
    uint8_t* st = lds + stage % S * T::STAGE;
#pragma unroll
    for (int i = 0; i < T::A_PER_WAVE; ++i) {
      const int c = wave * T::A_PER_WAVE + i, g = c / (BM / 8), kb = (stage * G + g) * kBlock;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr,
          (__attribute__((address_space(3))) void*)(st + T::SCALES + g * T::BLOCK + c % (BM / 8) * 1024),
          16, (int)(dslot < p.k - kb ? a_off[i] : kOutOfRange), kb, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < T::B_PER_WAVE; ++i) {
      const int c = wave * T::B_PER_WAVE + i, g = c / (BN / 8), kb = (stage * G + g) * kBlock;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr,
          (__attribute__((address_space(3))) void*)(st + T::SCALES + g * T::BLOCK + BM * kBlock +
                                                    c % (BN / 8) * 1024),
          16, (int)(dslot < p.k - kb ? b_off[i] : kOutOfRange), kb, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < T::S_PER_WAVE; ++i) {
      const int part = (wave * T::S_PER_WAVE + i) % T::SCALE_PARTS;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          sr, (__attribute__((address_space(3))) void*)(st + part * 256), 4,
          (int)(stage * G + s_block[i] < p.blocks ? s_off[i] : kOutOfRange),
          stage * G < p.blocks ? stage * G * (int)p.xs_block * 4 : 0, 0, 0);
    }
  };
  const int lr = lane & 15, lq = lane >> 4;
  const int rd0 = lr * kBlock + ((lq ^ (lr & 7)) * 16);
  const int rd1 = lr * kBlock + (((lq + 4) ^ (lr & 7)) * 16);
  const int a_base = T::SCALES + wm * TM * 16 * kBlock;
  const int b_base = T::SCALES + (BM + wn * TN * 16) * kBlock;
  const int s_base = (wm * TM * 16 + lr) * 4;
  const int64_t wcol = n0 + wn * TN * 16;
  const float* ws = p.ws + (wcol < p.n ? wcol / kBlock : 0) * p.ws_row;
  float w_scales = lane < p.blocks ? ws[lane] : 0.f;
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int stages = (p.blocks + G - 1) / G;
#pragma unroll
  for (int t = 0; t < S - 1; ++t) issue(t);
  asm volatile("" : "+v"(w_scales));  // waited for here, and not at every use in the loop
  for (int t = 0, t64 = 64 / G; t < stages; ++t) {
    if (t == t64) {
      w_scales = t * G + lane < p.blocks ? ws[t * G + lane] : 0.f;
      asm volatile("" : "+v"(w_scales));
      t64 += 64 / G;
    }
    // stage t has arrived in every wave, and every wave has read stage t - 1, whose place the next
    // one takes
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * T::PER_WAVE) : "memory");
    asm volatile("s_barrier" ::: "memory");
    issue(t + S - 1);
    const uint8_t* st = lds + t % S * T::STAGE;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float sw = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w_scales), (t * G + g) & 63));
      Operand<EXACT> bv[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        bv[j] = Operand<EXACT>(read_operand(st + g * T::BLOCK + b_base + j * 16 * kBlock, rd0, rd1));
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const Operand<EXACT> a(read_operand(st + g * T::BLOCK + a_base + i * 16 * kBlock, rd0, rd1));
        const float s = *reinterpret_cast<const float*>(st + s_base + (g * BM + i * 16) * 4) * sw;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const f32x4 part = block_product(bv[j], a);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[e], s, acc[i][j][e]);
        }
      }
    }
  }

  // lane: row lane % 16 of row tile i, columns 4 (lane / 16) .. + 3 of column tile j
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int64_t col = wcol + j * 16 + lq * 4;
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias) load_values(p.bias + col, p.n - col, b);
#pragma unroll
    for (int i = 0; i < TM; ++i)
      store_columns<EXACT>(p, m0 + (wm * TM + i) * 16 + lr, col, acc[i][j], b);
  }
}

template <int WM, int WN, int TM, int TN, int S, int G, bool EXACT>
int launch_ring(GemmParams p, hipStream_t stream) {
  using T = RingTile<WM, WN, TM, TN, S, G>;
  if (T::BM * p.x_stride >= (int64_t)kOutOfRange || T::BN * p.w_stride >= (int64_t)kOutOfRange)
    return OMNI_ERR_UNSUPPORTED;
  const int64_t rt = (p.rows + T::BM - 1) / T::BM, ct = (p.n + T::BN - 1) / T::BN;
  if (rt * ct > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  p.row_tiles = (int)rt;
  p.col_tiles = (int)ct;
  auto k = block_fp8_ring_kernel<WM, WN, TM, TN, S, G, EXACT>;
  static const bool raised = hipFuncSetAttribute((const void*)k,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 T::LDS) == hipSuccess;
  if (!raised) return OMNI_ERR_LAUNCH;
  hipLaunchKernelGGL(k, dim3((unsigned)(rt * ct)), dim3(64 * T::NW), T::LDS, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

// ------------------------------------------------------------------------------ few rows
//
// Up to 16 rows: the weight's bytes are the time, each read once. A workgroup takes 16 columns of all
// rows; its waves take K blocks in turn and load their operands straight into MFMA registers, UNROLL
// blocks of them in flight. The blocks' products meet in LDS and are added in the blocks' order, as
// every other tile adds them, so that a row's bits are the same in any batch (a sum per wave, joined
// at the end, took 0.1 us less at 8 blocks and 0.8 us less at 64). x is E4M3 rows, or (XT) float rows,
// whose groups each wave quantizes for itself: the bits of omni_block_quantize without its launch. There
// the chain bounds it (1 x 1024 -> 2048 4.1 us, of E4M3 rows 3.5): the two halves of a row's block are
// loaded under load_piece's branches, one complete before the other goes out, both before the
// weights are asked for.

// What a lane holds of a row's K block: bytes (values) 16 q .. 16 q + 15 and 64 + 16 q .. + 15.
template <typename XT>
struct RowPiece {
  XT v[2][16];
};

template <typename XT>
OMNI_DEVICE void load_piece(const XT* row, int valid, RowPiece<XT>* piece) {
  typedef XT vec __attribute__((ext_vector_type(16)));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const XT* src = row + h * 64;
    if (valid >= h * 64 + 16) {
      vec t;
      __builtin_memcpy(&t, src, sizeof(t));
#pragma unroll
      for (int e = 0; e < 16; ++e) piece->v[h][e] = t[e];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) piece->v[h][e] = h * 64 + e < valid ? src[e] : (XT)0.f;
    }
  }
}

// The operand bytes of a row piece and the row's scale: the four lanes lane % 16 + 16 q share a row.
template <typename XT>
OMNI_DEVICE i32x8 quantize_piece(const RowPiece<XT>& piece, float* scale) {
  float amax = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf((float)piece.v[h][e]));
  amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
  float unit;
  *scale = group_scale(amax, &unit);
  i32x8 bytes;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const XT* v = &piece.v[w / 4][w % 4 * 4];
    int b = 0;
    b = __builtin_amdgcn_cvt_pk_fp8_f32((float)v[0] * unit, (float)v[1] * unit, b, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32((float)v[2] * unit, (float)v[3] * unit, b, true);
    bytes[w] = b;
  }
  return bytes;
}

// LDS bytes of a K block's products and scales, and how many blocks' a workgroup takes at most (two
// workgroups a CU then; a second chunk waits for the first one's sums).
constexpr int kFewBlockBytes = 1024 + 64, kFewChunk = 64;

template <int NW, int UNROLL, bool EXACT, typename XT>
__global__ void __launch_bounds__(64 * NW) block_fp8_few_rows_kernel(const GemmParams p) {
  constexpr bool FLOATS = !std::is_same<XT, uint8_t>::value;
  static_assert(NW >= 8, "a wave for each block that fills up eight");
  extern __shared__ __attribute__((aligned(16))) f32x4 products[];     // [chunk][64 lanes]
  float* scales = reinterpret_cast<float*>(products + p.chunk * 64);  // [chunk][16 rows]
  const int rows = (int)p.rows;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int64_t n0 = (int64_t)xcd_tile(blockIdx.x, p.col_tiles) * 16;
  const int n_rows = (int)(p.n - n0 < 16 ? p.n - n0 : 16);
  const auto wr = buffer_rsrc(p.w + n0 * p.w_stride, (uint32_t)((n_rows - 1) * p.w_stride + p.k));
  const uint32_t w_off = lr < n_rows ? (uint32_t)(lr * (int)p.w_stride + lq * 16) : kOutOfRange;
  const auto xr = buffer_rsrc(p.x, FLOATS ? 0u : (uint32_t)((p.rows - 1) * p.x_stride + p.k));
  const float* ws = p.ws + n0 / kBlock * p.ws_row;
  const uint32_t x_off = lr < rows ? (uint32_t)(lr * (int)p.x_stride + lq * 16) : kOutOfRange;
  const float* xs = FLOATS ? nullptr : p.xs + (lr < rows ? lr : 0) * p.xs_row;

  // a piece past k (its 16 bytes all are) reads zeros, blocks past the last one too
  auto load16 = [&](__amdgpu_buffer_rsrc_t r, uint32_t off, int at) __attribute__((always_inline)) {
    return __builtin_bit_cast(
        i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at + lq * 16 < p.k ? off : kOutOfRange, at, 0));
  };
  // the sums: element threadIdx.x % 4 of lane threadIdx.x / 4, in the first four waves
  const int out_row = threadIdx.x >> 2 & 15;
  const int64_t col = n0 + (threadIdx.x >> 6) * 4 + (threadIdx.x & 3);
  float acc = 0.f;
  for (int c0 = 0; c0 < p.blocks; c0 += p.chunk) {
    const int held = p.blocks - c0 < p.chunk ? p.blocks - c0 : p.chunk;
    if (c0 > 0) __syncthreads();  // the products before these are added
    if (const int at = held + wave; at < (held + 7) / 8 * 8) {  // the sums take eight blocks at a time
      products[at * 64 + lane] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (lane < 16) scales[at * 16 + lane] = 0.f;
    }
    for (int at0 = wave; at0 < held; at0 += NW * UNROLL) {
      i32x4 wv[UNROLL][2], xv[UNROLL][2];
      RowPiece<XT> xf[FLOATS ? UNROLL : 1];
      float sw[UNROLL], sx[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int kt = c0 + at0 + u * NW, kb = kt * kBlock;
        wv[u][0] = load16(wr, w_off, kb);
        wv[u][1] = load16(wr, w_off, kb + 64);
        sw[u] = kt < p.blocks ? ws[kt] : 0.f;
        if constexpr (FLOATS) {
          const XT* src = reinterpret_cast<const XT*>(p.x) + lr * p.x_stride + kb + lq * 16;
          load_piece(src, lr < rows ? p.x_features - kb - lq * 16 : 0, &xf[u]);
        } else {
          xv[u][0] = load16(xr, x_off, kb);
          xv[u][1] = load16(xr, x_off, kb + 64);
          sx[u] = kt < p.blocks ? xs[kt * p.xs_block] : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const Operand<EXACT> b(__builtin_shufflevector(wv[u][0], wv[u][1], 0, 1, 2, 3, 4, 5, 6, 7));
        i32x8 bytes;
        if constexpr (FLOATS)
          bytes = quantize_piece(xf[u], &sx[u]);
        else
          bytes = __builtin_shufflevector(xv[u][0], xv[u][1], 0, 1, 2, 3, 4, 5, 6, 7);
        const f32x4 part = block_product(b, Operand<EXACT>(bytes));
        const int at = at0 + u * NW;
        if (u == 0 || at < held) {
          products[at * 64 + lane] = part;
          if (lq == 0) scales[at * 16 + lr] = sx[u] * sw[u];
        }
      }
    }
    __syncthreads();
    if (wave < 4) {
      const float* part = reinterpret_cast<const float*>(products) + threadIdx.x;
      const float* s = scales + out_row;
      for (int j0 = 0; j0 < held; j0 += 8, part += 8 * 256, s += 8 * 16)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc = __builtin_fmaf(part[j * 256], s[j * 16], acc);
    }
  }
  if (wave >= 4 || out_row >= rows || col >= p.n) return;
  const float v[1] = {acc + (p.bias ? p.bias[col] : 0.f)};
  const int64_t at = out_row * p.out_stride + col;
  if (!EXACT)
    store_values<__bf16, 1>(static_cast<__bf16*>(p.out) + at, 1, v);
  else if (p.out_dtype == OMNI_DTYPE_F32)
    store_values<float, 1>(static_cast<float*>(p.out) + at, 1, v);
  else
    store_values<_Float16, 1>(static_cast<_Float16*>(p.out) + at, 1, v);
}

template <int NW, int UNROLL, bool EXACT, typename XT>
int launch_few_rows(GemmParams p, hipStream_t stream) {
  // 8-bit rows are read through a buffer resource, float rows by their addresses
  constexpr bool FLOATS = !std::is_same<XT, uint8_t>::value;
  if ((!FLOATS && p.rows * p.x_stride >= (int64_t)kOutOfRange) ||
      16 * p.w_stride >= (int64_t)kOutOfRange || (p.n + 15) / 16 > 0x7fffffffLL)
    return OMNI_ERR_UNSUPPORTED;
  const int all = (p.blocks + 7) / 8 * 8;
  p.chunk = all < kFewChunk ? all : kFewChunk;
  p.col_tiles = (int)((p.n + 15) / 16);
  auto k = block_fp8_few_rows_kernel<NW, UNROLL, EXACT, XT>;
  static const bool raised = hipFuncSetAttribute((const void*)k,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 kFewChunk * kFewBlockBytes) == hipSuccess;
  if (!raised) return OMNI_ERR_LAUNCH;
  hipLaunchKernelGGL(k, dim3((unsigned)p.col_tiles), dim3(64 * NW),
                     (unsigned)(p.chunk * kFewBlockBytes), stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

// ------------------------------------------------------------------------------ quantize

// 16 lanes per group of 128, 8 values each: the group's largest magnitude over the 16 lanes, then
// the values times 448 / amax rounded once (to nearest even, as the hardware conversion does). One read
// and one write of the rows; at 773 x 1040 the launch's 3.5 us are its latency.
template <typename T>
__global__ void __launch_bounds__(256) block_quantize_kernel(const T* x, int64_t x_stride, int64_t rows, int k,
                                                             int padded, int groups, uint8_t* q,
                                                             int64_t q_stride, float* scale,
                                                             int64_t scale_stride) {
  const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  const int lane = threadIdx.x & 15;
  const int64_t row = group / groups;
  if (row >= rows) return;  // all 16 lanes of a group alike
  const int g = (int)(group - row * groups);
  const int c = g * kBlock + lane * 8;
  float v[8];
  load_values<T, 8>(x + row * x_stride + c, k - c, v);
  u32x2 packed;
  const float s = quantize_group(v, &packed);
  uint8_t* dst = q + row * q_stride + c;
  if (c < padded) *reinterpret_cast<u32x2*>(dst) = packed;
  if (lane == 0) scale[row * scale_stride + g] = s;
}

int quantize_rows(const void* x, int x_dtype, int64_t x_stride, int64_t rows, int64_t k, void* q,
                  int64_t q_stride, float* scale, int64_t scale_stride, hipStream_t s) {
  const int64_t padded = (k + 15) / 16 * 16, groups = (k + kBlock - 1) / kBlock;
  const int64_t workgroups = (rows * groups * 16 + 255) / 256;
  if (workgroups > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  auto go = [&](auto* src) -> int {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
    hipLaunchKernelGGL(block_quantize_kernel<T>, dim3((unsigned)workgroups), dim3(256), 0, s, src,
                       x_stride, rows, (int)k, (int)padded, (int)groups,
                       static_cast<uint8_t*>(q), q_stride, scale, scale_stride);
    OMNI_LAUNCH_CHECK();
    return OMNI_OK;
  };
  if (x_dtype == OMNI_DTYPE_F32) return go(static_cast<const float*>(x));
  if (x_dtype == OMNI_DTYPE_BF16) return go(static_cast<const __bf16*>(x));
  return go(static_cast<const _Float16*>(x));
}

bool float_rows(int dtype) {
  return dtype == OMNI_DTYPE_F32 || dtype == OMNI_DTYPE_BF16 || dtype == OMNI_DTYPE_F16;
}

// Compute units of the device, asked once per process; 256 (MI355X) when the query fails.
int compute_units() {
  static const int cached = [] {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        cus <= 0) {
      (void)hipGetLastError();
      return 256;
    }
    return cus;
  }();
  return cached;
}

// The tiles, and what a K block of one costs when every CU has `per_cu` of them, in us, with the
// rest of the call (launch, first loads, output): measured with 256 and 512 tiles at 8 and 48 blocks,
// weights from HBM. The second pair is the exact form's. A choice by these: rows x k -> n and us of
// the tiles on both sides of it, 64 x 4096 -> 4096: 32 x 32 9.5, 32 x 64 11.6; 128 x 4096 -> 4096:
// 32 x 64 11.6, 32 x 32 16.2 (two rounds); 256 x 4096 -> 4096: 64 x 64 16.4, 32 x 64 20.9; 768 x
// 1024 -> 6144: 128 x 128 12.4, 64 x 64 24.3; 8192 x 4096 -> 8192: 256 x 256 280, 128 x 128 344.
enum { kTile32x32, kTile32x64, kTile64x64, kTile64x128, kTile128x128, kTile256x256, kTiles };
struct TileCost {
  int rows, columns, per_cu;
  float block, rest, exact_block, exact_rest;
};
constexpr TileCost kTileCosts[kTiles] = {
    {32, 32, 1, 0.152f, 3.4f, 0.213f, 3.4f},   {32, 64, 1, 0.205f, 3.5f, 0.329f, 3.6f},
    {64, 64, 1, 0.370f, 3.5f, 0.473f, 4.4f},   {64, 128, 1, 0.547f, 3.8f, 0.792f, 4.9f},
    {128, 128, 2, 1.407f, 5.3f, 2.180f, 7.4f}, {256, 256, 1, 2.086f, 9.2f, 1e9f, 1e9f}};

int choose_tile(int64_t rows, int64_t n, int blocks, bool exact) {
  const int64_t cus = compute_units();
  int best = 0;
  float best_us = 0.f;
  for (int t = 0; t < kTiles; ++t) {
    const TileCost& c = kTileCosts[t];
    const int64_t tiles = ((rows + c.rows - 1) / c.rows) * ((n + c.columns - 1) / c.columns);
    const int64_t rounds = (tiles + cus * c.per_cu - 1) / (cus * c.per_cu);
    float block = exact ? c.exact_block : c.block;
    const float rest = exact ? c.exact_rest : c.rest;
    // a CU that gets one tile of two runs it in a little over half the time
    if (c.per_cu == 2 && tiles <= cus) block *= 0.55f;
    const float us = (float)rounds * ((float)blocks * block + rest - 2.5f);
    if (t == 0 || us < best_us) {
      best = t;
      best_us = us;
    }
  }
  return best;
}

template <bool EXACT>
int launch_tile(int tile, const GemmParams& p, hipStream_t s) {
  switch (tile) {
    case kTile32x32: return launch_ring<2, 2, 1, 1, 4, 4, EXACT>(p, s);
    case kTile32x64: return launch_ring<2, 4, 1, 1, 3, 4, EXACT>(p, s);
    case kTile64x64:
      // exact products widen each operand: fewer waves with larger parts widen fewer (0.47 us a block
      // against 0.54 on 8 waves; 8-bit products 0.37 on 8, 0.42 on 4)
      if constexpr (EXACT) return launch_ring<2, 2, 2, 2, 4, 2, true>(p, s);
      else return launch_ring<2, 4, 2, 1, 4, 2, false>(p, s);
    case kTile64x128: return launch_ring<2, 4, 2, 2, 3, 2, EXACT>(p, s);
    case kTile128x128: return launch_gemm<2, 2, 4, 4, EXACT>(p, s);
    default: break;
  }
  if constexpr (!EXACT) return launch_gemm<2, 4, 8, 4, false>(p, s);
  return OMNI_ERR_INVALID_ARG;  // no 256 x 256 form: its widened operands do not fit the registers
}

// Up to 16 rows: 8 waves of two blocks in flight each, or, quantizing float rows themselves, 16 of
// one (1 x 1024 -> 2048 3.5 us, 16 x 4096 -> 4096 8.2; 16 waves of one block 3.4 and 8.7; float rows
// 4.1 and 8.6, with 8 waves 4.1 and 10.4, quantized by a launch before 5.6 and 11.2).
template <bool EXACT>
int launch_few(int x_dtype, const GemmParams& p, hipStream_t s) {
  switch (x_dtype) {
    case OMNI_DTYPE_FP8_E4M3: return launch_few_rows<8, 2, EXACT, uint8_t>(p, s);
    case OMNI_DTYPE_F32: return launch_few_rows<16, 1, EXACT, float>(p, s);
    case OMNI_DTYPE_BF16: return launch_few_rows<16, 1, EXACT, __bf16>(p, s);
    default: return launch_few_rows<16, 1, EXACT, _Float16>(p, s);
  }
}

}  // namespace

extern "C" int omni_block_quantize(const void* x, int x_dtype, int64_t x_stride, int64_t rows,
                                   int64_t k, void* q, int64_t q_stride, float* scale,
                                   int64_t scale_stride, omni_stream_t stream) {
  if (rows < 0 || k < 1 || k > kMaxFeatures || !float_rows(x_dtype)) return OMNI_ERR_INVALID_ARG;
  if (rows == 0) return OMNI_OK;
  if (!x || !q || !scale || x_stride < k || q_stride < (k + 15) / 16 * 16 || q_stride % 16 ||
      scale_stride < (k + kBlock - 1) / kBlock || !aligned_to(q, 16) || !aligned_to(scale, 4) ||
      !aligned_to(x, x_dtype == OMNI_DTYPE_F32 ? 4 : 2))
    return OMNI_ERR_INVALID_ARG;
  return quantize_rows(x, x_dtype, x_stride, rows, k, q, q_stride, scale, scale_stride,
                       reinterpret_cast<hipStream_t>(stream));
}

extern "C" int omni_block_fp8_gemm(const omni_block_fp8_args* a, omni_stream_t stream) {
  if (!a || a->rows < 0 || a->n < 1 || a->k < 16 || a->k % 16 || a->k > kMaxFeatures)
    return OMNI_ERR_INVALID_ARG;
  const bool floats = float_rows(a->x_dtype);
  if (!floats && a->x_dtype != OMNI_DTYPE_FP8_E4M3) return OMNI_ERR_INVALID_ARG;
  if (!float_rows(a->out_dtype)) return OMNI_ERR_INVALID_ARG;
  if (a->rows == 0) return OMNI_OK;
  const int64_t blocks = (a->k + kBlock - 1) / kBlock;
  const int out_size = a->out_dtype == OMNI_DTYPE_F32 ? 4 : 2;
  if (!a->x || !a->w || !a->w_scale || !a->out || a->w_stride < a->k || a->w_stride % 16 ||
      !aligned_to(a->w, 16) || a->out_stride < a->n || a->w_scale_stride < blocks ||
      !aligned_to(a->w_scale, 4) || !aligned_to(a->bias, 4) || !aligned_to(a->out, out_size))
    return OMNI_ERR_INVALID_ARG;
  const bool few = a->rows <= OMNI_BLOCK_FP8_FEW_ROWS;
  if (floats) {
    if (a->features < 1 || (a->features + 15) / 16 * 16 != a->k || a->x_stride < a->features ||
        !aligned_to(a->x, a->x_dtype == OMNI_DTYPE_F32 ? 4 : 2))
      return OMNI_ERR_INVALID_ARG;
    if (!few && (!a->workspace || !aligned_to(a->workspace, 16) ||
                 a->workspace_bytes < a->rows * (a->k + blocks * 4)))
      return OMNI_ERR_INVALID_ARG;
  } else if (!a->x_scale || a->x_stride < a->k || a->x_stride % 16 || !aligned_to(a->x, 16) ||
             a->x_scale_stride_row < 0 || a->x_scale_stride_block < 0 || !aligned_to(a->x_scale, 4)) {
    return OMNI_ERR_INVALID_ARG;
  }
  GemmParams p{};
  p.x = static_cast<const uint8_t*>(a->x);
  p.x_stride = a->x_stride;
  p.x_features = (int)a->features;
  p.xs = a->x_scale;
  p.xs_row = a->x_scale_stride_row;
  p.xs_block = a->x_scale_stride_block;
  p.w = static_cast<const uint8_t*>(a->w);
  p.w_stride = a->w_stride;
  p.ws = a->w_scale;
  p.ws_row = a->w_scale_stride;
  p.rows = a->rows;
  p.n = a->n;
  p.k = (int)a->k;
  p.blocks = (int)blocks;
  p.bias = a->bias;
  p.out = a->out;
  p.out_stride = a->out_stride;
  p.out_dtype = a->out_dtype;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool exact = a->out_dtype != OMNI_DTYPE_BF16;
  if (few)
    return exact ? launch_few<true>(a->x_dtype, p, s) : launch_few<false>(a->x_dtype, p, s);
  // the DMAs address a tile's scales, up to those of the last block, with 32-bit byte offsets
  if (256 * p.xs_row + blocks * p.xs_block >= 0x1fffffffLL) return OMNI_ERR_UNSUPPORTED;
  if (floats) {
    uint8_t* q = static_cast<uint8_t*>(a->workspace);
    float* scale = reinterpret_cast<float*>(q + a->rows * a->k);
    const int rc = quantize_rows(a->x, a->x_dtype, a->x_stride, a->rows, a->features, q, a->k, scale,
                                 blocks, s);
    if (rc != OMNI_OK) return rc;
    p.x = q;
    p.x_stride = a->k;
    p.xs = scale;
    p.xs_row = blocks;
    p.xs_block = 1;
  }
  const int tile = choose_tile(p.rows, p.n, p.blocks, exact);
  return exact ? launch_tile<true>(tile, p, s) : launch_tile<false>(tile, p, s);
}
