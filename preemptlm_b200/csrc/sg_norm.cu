// Root-mean-square norm with the residual's addition, and bf16 rows in 8 bits
// with a scale for every 128 values.
#include "sg_fp8.cuh"

namespace sg {

// One CTA per row, the row in registers: h = x + residual, y = h * rsqrt(mean
// (h^2) + eps) * weight, all in fp32, rounded once where it is stored (h and y
// to bf16, or y to e4m3 with a scale per 128 values).  Thread i holds the
// 8-value chunks i, i + blockDim, ...; 16 neighbouring lanes hold one block of
// 128, so its largest magnitude is four shuffles.  Bound by the rows' bytes: 8192 x
// 4096 with the residual 41.8 us (268 MB, 6.4 TB/s, 0.98 of a copy's rate); one row is
// a chain of two latencies, 1.6 us.  One chunk a thread up to 2048 values (26 to 29
// registers, 8 CTAs of 256 on an SM), two up to 8192 (40: six CTAs of 256 at 4096
// values, three of 512 at 8192), four beyond (about 50: up to 1024 threads, one CTA).
template <int VPT, bool FP8>
__global__ void __launch_bounds__(256 * VPT)
add_rms_norm_kernel(const uint16_t* x, const uint16_t* residual,
                    const uint16_t* weight, int T, int H, float eps, uint16_t* h_out,
                    uint16_t* y, uint8_t* y8, float* scales) {
  __shared__ float part[32];
  wait_for_previous();
  const int nvec = H >> 3;
  const size_t row = blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * H);
  const uint4* rr = reinterpret_cast<const uint4*>(residual + row * H);
  uint4 xv[VPT], rv[VPT], wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    xv[i] = rv[i] = wv[i] = make_uint4(0, 0, 0, 0);
    if (v < nvec) {
      xv[i] = ld_stream_v4(xr + v);
      if (residual) rv[i] = ld_stream_v4(rr + v);
      if (VPT <= 2) wv[i] = *(reinterpret_cast<const uint4*>(weight) + v);  // four chunks' do not fit the registers
    }
  }
  float h[VPT][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    unpack8(xv[i], h[i]);
    if (residual) {
      float r[8];
      unpack8(rv[i], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] += r[j];
      const int v = i * blockDim.x + threadIdx.x;
      if (v < nvec) reinterpret_cast<uint4*>(h_out + row * H)[v] = pack8(h[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(h[i][j], h[i][j], ss);
  }
  ss = warp_fold_sum(ss);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
  if (nwarps > 1) {
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = warp_fold_sum(lane < nwarps ? part[lane] : 0.0f);
  }
  const float rstd = rsqrtf(ss / static_cast<float>(H) + eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    float w[8];
    if (VPT > 2 && v < nvec) wv[i] = *(reinterpret_cast<const uint4*>(weight) + v);
    unpack8(wv[i], w);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] *= h[i][j] * rstd;
    if constexpr (FP8) {
      float amax = 0.0f;  // chunks past the row's end hold zeros
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(w[j]));
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      const float s = fp8_block_scale(amax);
      if (v < nvec) {
        reinterpret_cast<uint2*>(y8 + row * H)[v] = fp8_pack8(w, s);
        if ((v & 15) == 0) scales[static_cast<size_t>(v >> 4) * T + row] = s;
      }
    } else {
      if (v < nvec) reinterpret_cast<uint4*>(y + row * H)[v] = pack8(w);
    }
  }
}

// Rows in 8 bits: one thread per 8 values, 16 lanes per block of 128.  Bound by the
// rows' bytes; a few hundred rows are one launch's latency (333 x 4096 about 2.5 us).
__global__ void __launch_bounds__(256)
quantize_fp8_kernel(const uint16_t* x, int T, int K, uint8_t* x8,
                    float* scales) {
  wait_for_previous();
  const int vecs = ((K + FP8_BLOCK - 1) / FP8_BLOCK) * (FP8_BLOCK / 8);  // chunks of a row, whole blocks
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long t = i / vecs;
  const int v = static_cast<int>(i - t * vecs);
  const bool in = t < T && v * 8 < K;
  float f[8];
  unpack8(in ? ld_stream_v4(x + t * K + v * 8) : make_uint4(0, 0, 0, 0), f);
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  const float s = fp8_block_scale(amax);
  if (!in) return;
  *reinterpret_cast<uint2*>(x8 + t * K + v * 8) = fp8_pack8(f, s);
  if ((v & 15) == 0) scales[static_cast<size_t>(v >> 4) * T + t] = s;
}

template <int VPT>
static cudaError_t launch_norm(const uint16_t* x, const uint16_t* residual, const uint16_t* weight, int T, int H, float eps,
                        uint16_t* h, uint16_t* y, uint8_t* y8, float* scales, cudaStream_t s) {
  const int threads = ((H / 8 + VPT - 1) / VPT + 31) / 32 * 32;
  return launch_after_previous(y8 ? add_rms_norm_kernel<VPT, true> : add_rms_norm_kernel<VPT, false>, T, threads, 0, s, x,
                               residual, weight, T, H, eps, h, y, y8, scales);
}

static bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace sg

extern "C" int sg_add_rms_norm(const uint16_t* x, const uint16_t* residual, const uint16_t* weight, int T, int H,
                               float eps, uint16_t* h, uint16_t* y, uint8_t* y8, float* scales, void* stream) {
  if (T < 0 || (residual == nullptr) != (h == nullptr)) return SG_ERR_INVALID_ARG;
  if ((y8 == nullptr) != (scales == nullptr) || (T > 0 && (y == nullptr) == (y8 == nullptr))) return SG_ERR_INVALID_ARG;
  if (H < 8 || H % 8 || H > 32768) return SG_ERR_SHAPE;
  if (T == 0) return SG_OK;
  if (!x || !weight) return SG_ERR_INVALID_ARG;
  if (sg::misaligned16(x) || sg::misaligned16(residual) || sg::misaligned16(weight) || sg::misaligned16(h) ||
      sg::misaligned16(y) || sg::misaligned16(y8))
    return SG_ERR_INVALID_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  const int nvec = H / 8;
  if (nvec <= 256) SG_CUDA_TRY(sg::launch_norm<1>(x, residual, weight, T, H, eps, h, y, y8, scales, s));
  else if (nvec <= 1024) SG_CUDA_TRY(sg::launch_norm<2>(x, residual, weight, T, H, eps, h, y, y8, scales, s));
  else SG_CUDA_TRY(sg::launch_norm<4>(x, residual, weight, T, H, eps, h, y, y8, scales, s));
  return SG_OK;
}

extern "C" int sg_quantize_fp8(const uint16_t* x, int T, int K, uint8_t* x8, float* scales, void* stream) {
  if (T < 0) return SG_ERR_INVALID_ARG;
  if (K < 8 || K % 8) return SG_ERR_SHAPE;
  if (T == 0) return SG_OK;
  if (!x || !x8 || !scales || sg::misaligned16(x) || sg::misaligned16(x8)) return SG_ERR_INVALID_ARG;
  const long long n = static_cast<long long>(T) * ((K + sg::FP8_BLOCK - 1) / sg::FP8_BLOCK) * (sg::FP8_BLOCK / 8);
  const long long blocks = (n + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return SG_ERR_SHAPE;
  SG_CUDA_TRY(sg::launch_after_previous(sg::quantize_fp8_kernel, (unsigned)blocks, 256, 0, (cudaStream_t)stream, x, T, K,
                                        x8, scales));
  return SG_OK;
}
