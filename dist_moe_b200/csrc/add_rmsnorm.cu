// The residual's addition and the RMS norm in front of a layer, forward and backward, with the output also as MXFP8 rows.
//
//   s = round_to_residual_type(x + r)          (without a residual: s = x)
//   y = bf16( s * rstd * (w + c) ),            rstd = rsqrt(mean(s^2) + eps)
// The norm is taken of the stored stream, so that the backward, which reads it back, differentiates the same values:
//   u = gy * (w + c),   gx = gr = gs + rstd * (u - s * rstd^2 * mean(u * s)),   gw = sum_t gy * s * rstd
// Quantised rows are those of the MXFP8 row quantiser applied to y, bit for bit, in the packed form that inference calls publish:
// D bytes E4M3, D / 32 scale bytes, padding to 16 bytes.
//
// HBM bound.  Rows of whole 16-byte pieces, up to 16384 values: every value stays in registers between its sum and its use, 2 + 2|4
// bytes in and 2 + 2|4 (+ 1.03) out per element, in the backward 2 + 2|4 + 2|4 in and 2 (+ 4) out.  A row belongs to a block of as many
// warps as it takes with two 16-byte pieces a lane (four beyond 8192 values); in the backward one of up to 1024 values to a warp, four
// pieces a lane, four rows to a block: 16384 rows of 256 and 1024 values took 28 and 47 us so, 36 and 50 with blocks (in the forward 15
// and 32 with warps, 15 and 30 with blocks).  The gain's gradient is summed over the rows of a block in registers and over the blocks
// by a second launch, always in the same order.
// All other rows go through forms of their own (add_rmsnorm_*_any_kernel): a value a load, rows read twice, and in the backward the
// gain's gradient of a block in memory, read and written for every row.  They take 1.4 to 2.4 times as long.
//
// Measured, L2 flushed, events included (some 6 us): 16384 x 4096 bf16 forward 94 us (5.7 TB/s), backward 116 us with the gain's gradient,
// 109 without; 4096 x 2816 with an fp32 stream 29 us, with quantised rows 31 us, backward 58 us (3.2 TB/s); 16384 x 1008 with a bf16 stream
// 31 and 48, fp32 37 and 79 (3.4 TB/s), and 16384 x 1001, the other form, 59 and 116, 55 and 144; 16 x 2048 8 us.
// What holds the backward at half of the copy rate where the stream is fp32 or a row a warp's: eight warps an SM in the warps' form, and
// the gain, which is the same for every row that a block walks over, loaded twice a row by every thread.
#include <type_traits>

#include "quant_common.cuh"
#include "../../include/dist_moe_b200.h"

namespace dm {

constexpr int kNormThreads = 512;              // of a row, at most
constexpr int kNormMaxVec = kNormThreads * 4;  // 16-byte pieces of bf16 that the register forms hold

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) { unpack8f(*reinterpret_cast<const uint4*>(p), f); }
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ float rounded(const __nv_bfloat16*, float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
__device__ __forceinline__ float rounded(const float*, float v) { return v; }

struct Gain {
  const void* w;
  int is_f32;
  float center;
  __device__ __forceinline__ void load(int64_t i, float (&g)[8]) const {
    if (is_f32)
      load8(static_cast<const float*>(w) + i, g);
    else
      load8(static_cast<const __nv_bfloat16*>(w) + i, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] += center;
  }
  __device__ __forceinline__ float at(int64_t i) const {
    return (is_f32 ? static_cast<const float*>(w)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i])) + center;
  }
};

struct QuantRows {
  uint8_t* rows;  // null: not wanted
  int64_t stride;
};

__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// Sum over a row's threads: a warp, or the whole block, whose `part` holds a word per warp.
template <bool kWarpRow>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = lanes_sum(v);
  if (kWarpRow) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  return lanes_sum(lane < warps ? part[lane] : 0.f);
}

// The E4M3 bytes and the scale of the block of 32 that four neighbouring lanes hold, 8 values each.  All lanes of a warp call.
__device__ __forceinline__ void quantise_piece(const uint4& y, int v, bool in, int64_t D, uint8_t* row) {
  uint32_t m = __vmaxu2(__vmaxu2(y.x & 0x7fff7fffu, y.y & 0x7fff7fffu), __vmaxu2(y.z & 0x7fff7fffu, y.w & 0x7fff7fffu));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  float recip;
  const uint32_t byte = mxfp8_scale_bits((m >> 16) > (m & 0xffffu) ? m >> 16 : m & 0xffffu, recip);
  if (!in) return;
  float f[8];
  unpack8f(y, f);
  *reinterpret_cast<uint2*>(row + static_cast<int64_t>(v) * 8) =
      make_uint2(e4m3x2_scaled(f[0], f[1], recip, recip) | (e4m3x2_scaled(f[2], f[3], recip, recip) << 16),
                 e4m3x2_scaled(f[4], f[5], recip, recip) | (e4m3x2_scaled(f[6], f[7], recip, recip) << 16));
  if ((v & 3) == 0) row[D + (v >> 2)] = static_cast<uint8_t>(byte);
}

// kVec pieces of 8 values a thread.
template <typename R, bool kResidual, int kVec>
__global__ void __launch_bounds__(kNormThreads) add_rmsnorm_fwd_kernel(
    const __nv_bfloat16* __restrict__ x, int64_t x_stride, const R* __restrict__ residual, int64_t r_stride, Gain gain, float eps,
    int vec, R* __restrict__ sum_out, __nv_bfloat16* __restrict__ y_out, float* __restrict__ rstd_out, QuantRows quant) {
  __shared__ float part[kNormThreads / 32];
  const int threads = blockDim.x, lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  const int64_t D = static_cast<int64_t>(vec) * 8;
  float s[kVec][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * threads + lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[i][j] = 0.f;
    if (v < vec) load8(x + t * x_stride + v * 8, s[i]);
  }
  if (kResidual) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = i * threads + lane;
      if (v < vec) {
        float r[8];
        load8(residual + t * r_stride + v * 8, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = rounded(residual, s[i][j] + r[j]);
        store8(sum_out + t * D + v * 8, s[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += s[i][j] * s[i][j];
  const float rstd = rsqrtf(row_sum<false>(ss, part) / static_cast<float>(D) + eps);
  if (rstd_out != nullptr && lane == 0) rstd_out[t] = rstd;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * threads + lane;
    const bool in = v < vec;
    uint4 y = make_uint4(0, 0, 0, 0);
    if (in) {
      float g[8];
      gain.load(v * 8, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = s[i][j] * rstd * g[j];
      y = make_uint4(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]), pack_bf16x2(g[6], g[7]));
      *reinterpret_cast<uint4*>(y_out + t * D + v * 8) = y;
    }
    if (quant.rows != nullptr) quantise_piece(y, v, in, D, quant.rows + t * quant.stride);
  }
  if (quant.rows != nullptr && lane < quant.stride - D - D / 32) quant.rows[t * quant.stride + D + D / 32 + lane] = 0;  // the row's padding
}

// Rows of any length, stride and alignment, a block each, read twice; not quantised.
template <typename R, bool kResidual>
__global__ void __launch_bounds__(256) add_rmsnorm_fwd_any_kernel(
    const __nv_bfloat16* __restrict__ x, int64_t x_stride, const R* __restrict__ residual, int64_t r_stride, Gain gain, float eps,
    int64_t T, int64_t D, R* sum_out, __nv_bfloat16* __restrict__ y_out, float* __restrict__ rstd_out) {
  __shared__ float part[8];
  const int64_t t = blockIdx.x;
  float ss = 0.f;
  for (int64_t i = threadIdx.x; i < D; i += 256) {
    float v = load1(x + t * x_stride + i);
    if (kResidual) {
      v = rounded(residual, v + load1(residual + t * r_stride + i));
      store1(sum_out + t * D + i, v);
    }
    ss += v * v;
  }
  const float rstd = rsqrtf(row_sum<false>(ss, part) / static_cast<float>(D) + eps);
  if (rstd_out != nullptr && threadIdx.x == 0) rstd_out[t] = rstd;
  for (int64_t i = threadIdx.x; i < D; i += 256) {  // each thread meets its own sums again
    const float v = kResidual ? load1(sum_out + t * D + i) : load1(x + t * x_stride + i);
    store1(y_out + t * D + i, v * rstd * gain.at(i));
  }
}

// A backward block keeps kStages rows (of four warps each its own) on their way in shared memory, as 16-byte pieces that the thread
// which asked for them reads back itself: no barrier stands between a copy and its use.  A row's arithmetic needs its sum first, so
// without the next rows on their way the loads stop for it.
template <typename R, int kVec>
struct NormBwd {
  static constexpr int kWide = sizeof(R) / 2;  // 16-byte pieces of eight values of the stream
  static constexpr int kPieces = kVec * (1 + 2 * kWide);
  static constexpr int stage_bytes(int threads) { return threads * kPieces * 16; }
  // Blocks of an SM: up to four.
  static constexpr int resident(int threads, int stages) {
    const int fit = 220 * 1024 / (stages * stage_bytes(threads) + 2048), most = kNormThreads * 2 / threads;
    return fit < 4 ? (fit < most ? fit : most) : (4 < most ? 4 : most);
  }
};

__device__ __forceinline__ void async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void unpack_wide(const uint4 (&v)[1], float (&f)[8]) { unpack8f(v[0], f); }
__device__ __forceinline__ void unpack_wide(const uint4 (&v)[2], float (&f)[8]) {
  const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
}

// Blocks walk over the rows, the next ones on their way; `partial` [gridDim.x][D] takes each block's share of the gain's gradient.
template <typename R, bool kWarpRow, int kVec, int kStages>
__global__ void __launch_bounds__(kWarpRow ? 128 : kNormThreads) add_rmsnorm_bwd_kernel(
    const __nv_bfloat16* __restrict__ grad_y, const R* __restrict__ grad_sum, const R* __restrict__ sum, int64_t sum_stride,
    Gain gain, const float* __restrict__ rstd_in, int64_t T, int vec, __nv_bfloat16* __restrict__ grad_x,
    float* __restrict__ grad_residual, float* __restrict__ partial) {
  constexpr int kRows = kWarpRow ? 4 : 1, kWide = NormBwd<R, kVec>::kWide, kPieces = NormBwd<R, kVec>::kPieces;
  extern __shared__ __align__(16) uint8_t norm_smem[];
  __shared__ float part[2][kNormThreads / 32];
  const int threads = kWarpRow ? 32 : blockDim.x, lane = kWarpRow ? threadIdx.x & 31 : threadIdx.x, slot = kWarpRow ? threadIdx.x >> 5 : 0;
  const int64_t D = static_cast<int64_t>(vec) * 8, step = static_cast<int64_t>(gridDim.x) * kRows;
  const uint32_t own = smem_u32(norm_smem) + threadIdx.x * 16;
  const uint32_t piece = blockDim.x * 16, stage_bytes = piece * kPieces;  // bytes between a thread's pieces, and between stages
  auto ask = [&](int64_t t, int stage) {
    if (t < T) {
      const uint32_t to = own + stage * stage_bytes;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const int v = i * threads + lane;
        if (v < vec) {
          async16(to + i * piece, grad_y + t * D + v * 8);
#pragma unroll
          for (int w = 0; w < kWide; ++w) {
            async16(to + (kVec + i * kWide + w) * piece, sum + t * sum_stride + v * 8 + w * (8 / kWide));
            if (grad_sum != nullptr) async16(to + (kVec * (1 + kWide) + i * kWide + w) * piece, grad_sum + t * D + v * 8 + w * (8 / kWide));
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float gw[kVec][8];
#pragma unroll
  for (int i = 0; i < kVec; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) gw[i][j] = 0.f;
  int64_t t = static_cast<int64_t>(blockIdx.x) * kRows + slot;
#pragma unroll
  for (int s = 0; s < kStages; ++s) ask(t + s * step, s);
  int it = 0, stage = 0;
  for (; t < T; t += step, ++it) {
    const float rstd = rstd_in[t];
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    uint4 gy[kVec], s[kVec][kWide], gs[kVec][kWide];
    const uint32_t at = own + stage * stage_bytes;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const bool in = i * threads + lane < vec;
      gy[i] = in ? shared16(at + i * piece) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWide; ++w) {
        s[i][w] = in ? shared16(at + (kVec + i * kWide + w) * piece) : make_uint4(0, 0, 0, 0);
        gs[i][w] = in && grad_sum != nullptr ? shared16(at + (kVec * (1 + kWide) + i * kWide + w) * piece) : make_uint4(0, 0, 0, 0);
      }
    }
    ask(t + kStages * step, stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = i * threads + lane;
      if (v < vec) {
        float g[8], a[8], y[8];
        gain.load(v * 8, g);
        unpack_wide(s[i], a);
        unpack8f(gy[i], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          gw[i][j] += y[j] * (a[j] * rstd);
          dot += y[j] * g[j] * a[j];
        }
      }
    }
    const float mean = row_sum<kWarpRow>(dot, part[it & 1]) / static_cast<float>(D) * (rstd * rstd);
    if (grad_x == nullptr && grad_residual == nullptr) continue;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = i * threads + lane;
      if (v < vec) {
        float g[8], a[8], y[8], o[8];
        gain.load(v * 8, g);
        unpack_wide(s[i], a);
        unpack8f(gy[i], y);
        unpack_wide(gs[i], o);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += rstd * (y[j] * g[j] - a[j] * mean);
        if (grad_x != nullptr) store8(grad_x + t * D + v * 8, o);
        if (grad_residual != nullptr) store8(grad_residual + t * D + v * 8, o);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (partial == nullptr) return;
  float* rows = reinterpret_cast<float*>(norm_smem);  // [kRows][32 * 8]
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * threads + lane;
    if (kRows > 1) {  // the block's warps in order
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) rows[(slot * 32 + lane) * 8 + j] = gw[i][j];
      __syncthreads();
      if (slot == 0)
#pragma unroll
        for (int r = 1; r < kRows; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) gw[i][j] += rows[(r * 32 + lane) * 8 + j];
    }
    if (slot == 0 && v < vec) store8(partial + blockIdx.x * D + v * 8, gw[i]);
  }
}

template <typename R>
__global__ void __launch_bounds__(256) add_rmsnorm_bwd_any_kernel(
    const __nv_bfloat16* __restrict__ grad_y, const R* __restrict__ grad_sum, const R* __restrict__ sum, int64_t sum_stride,
    Gain gain, const float* __restrict__ rstd_in, int64_t T, int64_t D, __nv_bfloat16* __restrict__ grad_x,
    float* __restrict__ grad_residual, float* partial) {
  __shared__ float part[2][8];
  int it = 0;
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x, ++it) {
    const float rstd = rstd_in[t];
    float dot = 0.f;
    for (int64_t i = threadIdx.x; i < D; i += 256) {
      const float g = load1(grad_y + t * D + i), s = load1(sum + t * sum_stride + i);
      dot += g * gain.at(i) * s;
      if (partial != nullptr) {  // a thread's own columns
        float* own = partial + blockIdx.x * D + i;
        *own = (it == 0 ? 0.f : *own) + g * (s * rstd);
      }
    }
    const float mean = row_sum<false>(dot, part[it & 1]) / static_cast<float>(D) * (rstd * rstd);
    if (grad_x == nullptr && grad_residual == nullptr) continue;
    for (int64_t i = threadIdx.x; i < D; i += 256) {
      const float g = load1(grad_y + t * D + i) * gain.at(i), s = load1(sum + t * sum_stride + i);
      const float v = (grad_sum != nullptr ? load1(grad_sum + t * D + i) : 0.f) + rstd * (g - s * mean);
      if (grad_x != nullptr) store1(grad_x + t * D + i, v);
      if (grad_residual != nullptr) grad_residual[t * D + i] = v;
    }
  }
}

// Sum of the blocks' shares: 32 columns a block, 32 warps that take every 32nd share and meet in order.
template <typename W>
__global__ void __launch_bounds__(1024) add_rmsnorm_gain_kernel(const float* __restrict__ partial, int shares, int64_t D, W* __restrict__ out) {
  __shared__ float part[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.f;
  if (c < D)
#pragma unroll 8
    for (int b = warp; b < shares; b += 32) sum += partial[b * D + c];
  part[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || c >= D) return;
#pragma unroll
  for (int w = 1; w < 32; ++w) sum += part[w][lane];
  store1(out + c, sum);
}

// Packed MXFP8 rows back to bf16, a warp a row: 4 significant bits times a power of two, exact down to bf16's smallest values.
__global__ void __launch_bounds__(256) mxfp8_dequant_rows_kernel(const uint8_t* __restrict__ rows, int64_t stride, int64_t T, int blocks_of_32,
                                                                 uint4* __restrict__ out) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (t >= T) return;
  const uint8_t* row = rows + t * stride;
  uint4* to = out + t * blocks_of_32 * 4;
#pragma unroll 4
  for (int v = threadIdx.x & 31; v < blocks_of_32 * 2; v += 32) {  // 16 values
    const uint4 q = reinterpret_cast<const uint4*>(row)[v];
    const uint32_t byte = row[blocks_of_32 * 32 + (v >> 1)];
    const float scale = byte == 0xffu ? __int_as_float(0x7fc00000) : byte == 0 ? 0x1p-127f : __uint_as_float(byte << 23);
    const uint32_t in[4] = {q.x, q.y, q.z, q.w};
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((in[j >> 1] >> (16 * (j & 1))) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      w[j] = pack_bf16x2(f.x * scale, f.y * scale);
    }
    to[2 * v] = make_uint4(w[0], w[1], w[2], w[3]);
    to[2 * v + 1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Blocks of the backward: as many as the device holds at once, so that few shares of the gain's gradient are left.
static int64_t norm_bwd_blocks(int64_t T, int64_t rows, int resident) {
  const int64_t most = grid_cap(resident), blocks = ceil_div64(T, rows);
  return blocks < most ? blocks : most;
}
constexpr int kNormAnyResident = 4;
static int norm_threads(int vec, int per_thread) { return (vec + 32 * per_thread - 1) / (32 * per_thread) * 32; }

}  // namespace dm

using namespace dm;

template <typename R, bool kResidual>
static int add_rmsnorm_fwd(const void* x, int64_t x_stride, const void* residual, int64_t r_stride, const Gain& gain, float eps,
                           int64_t T, int64_t D, void* sum_out, void* y_out, float* rstd_out, const QuantRows& quant, cudaStream_t st) {
  const auto* xp = static_cast<const __nv_bfloat16*>(x);
  const auto* rp = static_cast<const R*>(residual);
  auto* sp = static_cast<R*>(sum_out);
  auto* yp = static_cast<__nv_bfloat16*>(y_out);
  const bool vectors = D % 8 == 0 && D / 8 <= kNormMaxVec && aligned16(x) && x_stride % 8 == 0 && aligned16(gain.w) && aligned16(y_out) &&
                       (!kResidual || (aligned16(residual) && aligned16(sum_out) && r_stride % 8 == 0));
  if (!vectors) {
    if (quant.rows != nullptr) return kRcUnsupportedShape;
    add_rmsnorm_fwd_any_kernel<R, kResidual><<<static_cast<unsigned>(T), 256, 0, st>>>(xp, x_stride, rp, r_stride, gain, eps, T, D, sp, yp, rstd_out);
    return static_cast<int>(cudaGetLastError());
  }
  const int vec = static_cast<int>(D / 8);
  auto run = [&](auto kernel, int threads) {
    kernel<<<static_cast<unsigned>(T), threads, 0, st>>>(xp, x_stride, rp, r_stride, gain, eps, vec, sp, yp, rstd_out, quant);
    return static_cast<int>(cudaGetLastError());
  };
  if (vec <= 2 * kNormThreads) return run(add_rmsnorm_fwd_kernel<R, kResidual, 2>, norm_threads(vec, 2));
  return run(add_rmsnorm_fwd_kernel<R, kResidual, 4>, norm_threads(vec, 4));
}

extern "C" int dm_add_rmsnorm_fwd(const void* x, int64_t x_stride, const void* residual, int residual_is_f32, int64_t residual_stride,
                                  const void* weight, int weight_is_f32, float gain_center, float eps, int64_t T, int64_t D,
                                  void* sum_out, void* y_out, float* rstd_out, void* rows_out, int64_t row_stride, void* stream) {
  if (T < 0 || T > 0x7fffffff || D <= 0 || x_stride < 0 || residual_stride < 0) return kRcBadArg;
  if (T == 0) return kRcOk;
  if (!x || !weight || !y_out || (residual != nullptr) != (sum_out != nullptr)) return kRcBadArg;
  if (rows_out != nullptr && (D % 32 != 0 || row_stride % 16 != 0 || row_stride < D + D / 32 || row_stride >= D + D / 32 + 16 || !aligned16(rows_out)))
    return kRcUnsupportedShape;
  const Gain gain{weight, weight_is_f32, gain_center};
  const QuantRows quant{static_cast<uint8_t*>(rows_out), row_stride};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (residual == nullptr)
    return add_rmsnorm_fwd<__nv_bfloat16, false>(x, x_stride, nullptr, 0, gain, eps, T, D, nullptr, y_out, rstd_out, quant, st);
  if (residual_is_f32)
    return add_rmsnorm_fwd<float, true>(x, x_stride, residual, residual_stride, gain, eps, T, D, sum_out, y_out, rstd_out, quant, st);
  return add_rmsnorm_fwd<__nv_bfloat16, true>(x, x_stride, residual, residual_stride, gain, eps, T, D, sum_out, y_out, rstd_out, quant, st);
}

// An upper bound over the forms below.
extern "C" int64_t dm_add_rmsnorm_shares(int64_t T, int64_t D) { return T <= 0 || D <= 0 ? 0 : norm_bwd_blocks(T, 1, 4); }

template <typename R>
static int add_rmsnorm_bwd(const void* grad_y, const void* grad_sum, const void* sum, int64_t sum_stride, const Gain& gain,
                           const float* rstd, int64_t T, int64_t D, void* grad_x, float* grad_residual, float* partial, int& blocks,
                           cudaStream_t st) {
  const auto* gy = static_cast<const __nv_bfloat16*>(grad_y);
  const auto* gs = static_cast<const R*>(grad_sum);
  const auto* sp = static_cast<const R*>(sum);
  auto* gx = static_cast<__nv_bfloat16*>(grad_x);
  const bool vectors = D % 8 == 0 && D / 8 <= kNormMaxVec && aligned16(gy) && aligned16(gs) && aligned16(sp) && sum_stride % 8 == 0 &&
                       aligned16(gain.w) && aligned16(gx) && aligned16(grad_residual) && aligned16(partial);
  if (!vectors) {
    blocks = static_cast<int>(norm_bwd_blocks(T, 1, kNormAnyResident));
    add_rmsnorm_bwd_any_kernel<R><<<blocks, 256, 0, st>>>(gy, gs, sp, sum_stride, gain, rstd, T, D, gx, grad_residual, partial);
    return static_cast<int>(cudaGetLastError());
  }
  const int vec = static_cast<int>(D / 8);
  auto launch = [&](auto warp_tag, auto vec_tag, auto stages_tag, int threads) {
    constexpr bool warp_row = decltype(warp_tag)::value;
    constexpr int per_thread = decltype(vec_tag)::value, stages = decltype(stages_tag)::value;
    constexpr auto kernel = add_rmsnorm_bwd_kernel<R, warp_row, per_thread, stages>;
    static PerDeviceOnce attr_set;
    const int rc = once_per_device(
        attr_set, [] { return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 218 * 1024)); });
    if (rc != 0) return rc;
    using C = NormBwd<R, per_thread>;
    blocks = static_cast<int>(norm_bwd_blocks(T, warp_row ? 4 : 1, C::resident(threads, stages)));
    kernel<<<blocks, threads, stages * C::stage_bytes(threads), st>>>(gy, gs, sp, sum_stride, gain, rstd, T, vec, gx, grad_residual, partial);
    return static_cast<int>(cudaGetLastError());
  };
  using std::integral_constant;
  // Two stages (three were not faster), or one where they do not fit: rows of more than 10240 values with an fp32 stream.
  auto run = [&](auto warp_tag, auto vec_tag, int threads) {
    using C = NormBwd<R, decltype(vec_tag)::value>;
    constexpr bool always_fit = C::resident(decltype(warp_tag)::value ? 128 : kNormThreads, 2) >= 1;
    if constexpr (!always_fit)
      if (C::resident(threads, 2) < 1) return launch(warp_tag, vec_tag, integral_constant<int, 1>{}, threads);
    return launch(warp_tag, vec_tag, integral_constant<int, 2>{}, threads);
  };
  if (D <= 1024) return run(std::true_type{}, integral_constant<int, 4>{}, 128);
  if (vec <= 2 * kNormThreads) return run(std::false_type{}, integral_constant<int, 2>{}, norm_threads(vec, 2));
  return run(std::false_type{}, integral_constant<int, 4>{}, norm_threads(vec, 4));
}

extern "C" int dm_add_rmsnorm_bwd(const void* grad_y, const void* grad_sum, const void* sum, int sum_is_f32, int64_t sum_stride,
                                  const void* weight, int weight_is_f32, float gain_center, const float* rstd, int64_t T, int64_t D,
                                  void* grad_x, float* grad_residual, float* partial, void* grad_weight, void* stream) {
  if (T <= 0 || T > 0x7fffffff || D <= 0 || sum_stride < 0) return kRcBadArg;
  if (!grad_y || !sum || !weight || !rstd || (partial != nullptr) != (grad_weight != nullptr)) return kRcBadArg;
  const Gain gain{weight, weight_is_f32, gain_center};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int shares = 0;
  const int rc = sum_is_f32 ? add_rmsnorm_bwd<float>(grad_y, grad_sum, sum, sum_stride, gain, rstd, T, D, grad_x, grad_residual, partial, shares, st)
                            : add_rmsnorm_bwd<__nv_bfloat16>(grad_y, grad_sum, sum, sum_stride, gain, rstd, T, D, grad_x, grad_residual, partial,
                                                             shares, st);
  if (rc != 0 || grad_weight == nullptr) return rc;
  const unsigned columns = static_cast<unsigned>(ceil_div64(D, 32));
  if (weight_is_f32)
    add_rmsnorm_gain_kernel<float><<<columns, 1024, 0, st>>>(partial, shares, D, static_cast<float*>(grad_weight));
  else
    add_rmsnorm_gain_kernel<__nv_bfloat16><<<columns, 1024, 0, st>>>(partial, shares, D, static_cast<__nv_bfloat16*>(grad_weight));
  return static_cast<int>(cudaGetLastError());
}

extern "C" int dm_dequant_mxfp8_rows(const void* rows, int64_t row_stride, int64_t T, int64_t D, void* out, void* stream) {
  if (T < 0 || T > 0x7fffffff || D <= 0 || D % 32 != 0 || row_stride % 16 != 0 || row_stride < D + D / 32) return kRcBadArg;
  if (T == 0) return kRcOk;
  if (!rows || !out || !aligned16(rows) || !aligned16(out)) return kRcBadArg;
  mxfp8_dequant_rows_kernel<<<static_cast<unsigned>(ceil_div64(T, 8)), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(rows), row_stride, T, static_cast<int>(D / 32), static_cast<uint4*>(out));
  return static_cast<int>(cudaGetLastError());
}
