// Linear layers in 8-bit floating point (OCP E4M3) with a float32 scale for each block of 128:
//
//   y[m][n] = sum_b sx[m][b] * sw[n / 128][b] * (sum_{k in block b} x[m][k] * w[n][k]) (+ bias[n])
//
// block b holds k = 128 b .. 128 b + 127 (the last one shorter), and omni_block_quantize, which
// makes such rows from bf16 / f16 / float32 ones.
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
  const float* bias;
  void* out;
  int64_t out_stride;
  int out_dtype;
  int row_tiles, col_tiles;
};

// A tile of the output by WM x WN waves, each TM x TN MFMA tiles of 16 x 16. A K block's product
// starts from zero, and one fma per element adds it, scaled, to the float32 accumulator. Rows of 128 bytes travel to LDS by DMA into a ring of S stages; a
// row's 16-byte slot s is stored at s ^ (row % 8), so that the operand reads of 16 rows spread over
// all banks. A lane's 32 bytes of a row are slots q and q + 4 (q = lane / 16) for both operands, so
// the products of a block pair up whatever order the instruction numbers them in.
template <int WM, int WN, int TM, int TN, int S, bool EXACT>
__global__ void __launch_bounds__(64 * WM * WN) block_fp8_gemm_kernel(const GemmParams p) {
  constexpr int NW = WM * WN;
  constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
  constexpr int A_PER_WAVE = BM / 8 / NW, B_PER_WAVE = BN / 8 / NW;
  static_assert(BM / 8 % NW == 0 && BN / 8 % NW == 0 && TN * 16 <= 128, "tile split");
  constexpr int STAGE = (BM + BN) * kBlock;
  constexpr int PER_WAVE = A_PER_WAVE + B_PER_WAVE;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int tile = xcd_tile(blockIdx.x, p.row_tiles * p.col_tiles);
  const int ct = tile / p.row_tiles;
  const int64_t m0 = (int64_t)(tile - ct * p.row_tiles) * BM;
  const int64_t n0 = (int64_t)ct * BN;

  // resources of the tile's own rows: rows past the last read zeros
  const int64_t m_rows = p.rows - m0 < BM ? p.rows - m0 : BM;
  const int64_t n_rows = p.n - n0 < BN ? p.n - n0 : BN;
  const auto xr = buffer_rsrc(p.x + m0 * p.x_stride, (uint32_t)((m_rows - 1) * p.x_stride + p.k));
  const auto wr = buffer_rsrc(p.w + n0 * p.w_stride, (uint32_t)((n_rows - 1) * p.w_stride + p.k));
  const int drow = lane >> 3;
  const int dslot = ((lane & 7) ^ drow) * 16;  // the byte of the row this lane's DMA piece holds
  uint32_t a_off[A_PER_WAVE], b_off[B_PER_WAVE];
#pragma unroll
  for (int i = 0; i < A_PER_WAVE; ++i) {
    const int row = (wave * A_PER_WAVE + i) * 8 + drow;
    a_off[i] = row < m_rows ? (uint32_t)(row * (int)p.x_stride + dslot) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < B_PER_WAVE; ++i) {
    const int row = (wave * B_PER_WAVE + i) * 8 + drow;
    b_off[i] = row < n_rows ? (uint32_t)(row * (int)p.w_stride + dslot) : kOutOfRange;
  }
  auto issue = [&](int kt) __attribute__((always_inline)) {
    uint8_t* st = lds + (kt % S) * STAGE;
    const int kb = kt * kBlock;
    const bool in = dslot < p.k - kb;  // the last block may end early
#pragma unroll
    for (int i = 0; i < A_PER_WAVE; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (__attribute__((address_space(3))) void*)(st + (wave * A_PER_WAVE + i) * 1024), 16,
          (int)(in ? a_off[i] : kOutOfRange), kb, 0, 0);
#pragma unroll
    for (int i = 0; i < B_PER_WAVE; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr,
          (__attribute__((address_space(3))) void*)(st + BM * kBlock + (wave * B_PER_WAVE + i) * 1024),
          16, (int)(in ? b_off[i] : kOutOfRange), kb, 0, 0);
  };

  const int lr = lane & 15, lq = lane >> 4;
  const int rd0 = lr * kBlock + ((lq ^ (lr & 7)) * 16);
  const int rd1 = lr * kBlock + (((lq + 4) ^ (lr & 7)) * 16);
  const int a_base = wm * TM * 16 * kBlock;
  const int b_base = (BM + wn * TN * 16) * kBlock;

  // the scales of this lane's rows (row lane % 16 of each row tile) and of the wave's columns,
  // which lie in one block of 128
  const float* xs[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = m0 + (wm * TM + i) * 16 + lr;
    xs[i] = p.xs + (row < p.rows ? row : p.rows - 1) * p.xs_row;
  }
  const int64_t wcol = n0 + wn * TN * 16;
  const float* ws = p.ws + (wcol < p.n ? wcol / kBlock : 0) * p.ws_row;

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int kt = 0; kt < S - 1; ++kt)
    if (kt < p.blocks) issue(kt);
  for (int kt = 0; kt < p.blocks; ++kt) {
    float s[TM];
    const float sw = ws[kt];
#pragma unroll
    for (int i = 0; i < TM; ++i) s[i] = xs[i][kt * p.xs_block] * sw;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (kt + S - 1 < p.blocks) issue(kt + S - 1);
    const uint8_t* st = lds + (kt % S) * STAGE;
    Operand<EXACT> bv[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) 
      bv[j] = Operand<EXACT>(read_operand(st + b_base + j * 16 * kBlock, rd0, rd1));
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const Operand<EXACT> av(read_operand(st + a_base + i * 16 * kBlock, rd0, rd1));
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const f32x4 part = block_product(bv[j], av);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[e], s[i], acc[i][j][e]);
      }
    }
  }

  // lane: row lane % 16 of row tile i, columns 4 (lane / 16) .. + 3 of column tile j
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = m0 + (wm * TM + i) * 16 + lr;
#pragma unroll
    for (int j = 0; j < TN; ++j)
      store_columns(p.out, p.out_dtype, p.out_stride, p.bias, row, p.rows,
                    wcol + j * 16 + lq * 4, p.n, acc[i][j]);
  }
}

template <int WM, int WN, int TM, int TN, int S, bool EXACT>
int launch_gemm(GemmParams p, hipStream_t stream) {
  constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
  constexpr int lds_bytes = S * (BM + BN) * kBlock;
  if (BM * p.x_stride >= (int64_t)kOutOfRange || BN * p.w_stride >= (int64_t)kOutOfRange)
    return OMNI_ERR_UNSUPPORTED;
  const int64_t rt = (p.rows + BM - 1) / BM, ct = (p.n + BN - 1) / BN;
  if (rt * ct > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  p.row_tiles = (int)rt;
  p.col_tiles = (int)ct;
  auto k = block_fp8_gemm_kernel<WM, WN, TM, TN, S, EXACT>;
  static const bool raised = hipFuncSetAttribute((const void*)k,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 lds_bytes) == hipSuccess;
  if (!raised) return OMNI_ERR_LAUNCH;
  hipLaunchKernelGGL(k, dim3((unsigned)(rt * ct)), dim3(64 * WM * WN), lds_bytes, stream, p);
  OMNI_LAUNCH_CHECK();
  return OMNI_OK;
}

// ------------------------------------------------------------------------------ quantize

// 16 lanes per group of 128, 8 values each: the group's largest magnitude over the 16 lanes, then
// the values times 448 / amax rounded once (to nearest even, as the hardware conversion does).
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

}  // namespace

extern "C" int omni_block_quantize(const void* x, int x_dtype, int64_t x_stride, int64_t rows,
                                   int64_t k, void* q, int64_t q_stride, float* scale,
                                   int64_t scale_stride, omni_stream_t stream) {
  if (rows < 0 || k < 1 || k > kMaxFeatures) return OMNI_ERR_INVALID_ARG;
  if (rows == 0) return OMNI_OK;
  const int64_t padded = (k + 15) / 16 * 16, groups = (k + kBlock - 1) / kBlock;
  if (!x || !q || !scale || x_stride < k || q_stride < padded || q_stride % 16 ||
      scale_stride < groups || !aligned_to(q, 16) || !aligned_to(scale, 4))
    return OMNI_ERR_INVALID_ARG;
  const int64_t workgroups = (rows * groups * 16 + 255) / 256;
  if (workgroups > 0x7fffffffLL) return OMNI_ERR_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto* src) -> int {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
    if (!aligned_to(src, sizeof(T))) return OMNI_ERR_INVALID_ARG;
    hipLaunchKernelGGL(block_quantize_kernel<T>, dim3((unsigned)workgroups), dim3(256), 0, s, src,
                       x_stride, rows, (int)k, (int)padded, (int)groups,
                       static_cast<uint8_t*>(q), q_stride, scale, scale_stride);
    OMNI_LAUNCH_CHECK();
    return OMNI_OK;
  };
  switch (x_dtype) {
    case OMNI_DTYPE_F32: return go(static_cast<const float*>(x));
    case OMNI_DTYPE_BF16: return go(static_cast<const __bf16*>(x));
    case OMNI_DTYPE_F16: return go(static_cast<const _Float16*>(x));
    default: return OMNI_ERR_INVALID_ARG;
  }
}

extern "C" int omni_block_fp8_gemm(const omni_block_fp8_args* a, omni_stream_t stream) {
  if (!a || a->rows < 0 || a->n < 1 || a->k < 16 || a->k % 16 || a->k > kMaxFeatures)
    return OMNI_ERR_INVALID_ARG;
  if (a->rows == 0) return OMNI_OK;
  const int64_t blocks = (a->k + kBlock - 1) / kBlock;
  const int64_t out_size = a->out_dtype == OMNI_DTYPE_F32 ? 4 : 2;
  if (!a->x || !a->x_scale || !a->w || !a->w_scale || !a->out || a->x_stride < a->k ||
      a->w_stride < a->k || a->x_stride % 16 || a->w_stride % 16 || !aligned_to(a->x, 16) ||
      !aligned_to(a->w, 16) || a->out_stride < a->n || a->x_scale_stride_row < 0 ||
      a->x_scale_stride_block < 0 || a->w_scale_stride < blocks || !aligned_to(a->x_scale, 4) ||
      !aligned_to(a->w_scale, 4) || !aligned_to(a->bias, 4) || !aligned_to(a->out, (int)out_size))
    return OMNI_ERR_INVALID_ARG;
  if (a->out_dtype != OMNI_DTYPE_F32 && a->out_dtype != OMNI_DTYPE_BF16 &&
      a->out_dtype != OMNI_DTYPE_F16)
    return OMNI_ERR_INVALID_ARG;
  GemmParams p{};
  p.x = static_cast<const uint8_t*>(a->x);
  p.x_stride = a->x_stride;
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
  return a->out_dtype == OMNI_DTYPE_BF16 ? launch_gemm<2, 2, 2, 2, 2, false>(p, s)
                                         : launch_gemm<2, 2, 2, 2, 2, true>(p, s);
}
