// RMS norm with the residual's addition in front and the 1 x 128 e4m3 quantiser behind: what enters an FP8 Linear.
//
//   h = round(x + residual)   y = h * rsqrt(mean(h^2) + eps) * (w + offset)   s = amax_128(|y|) / 448   y8 = e4m3(y / s)
//
// One pass: a block owns a row, its 16-byte chunks of h stay packed in registers between the two reductions (sum of
// squares over the row, |y| maximum over the 16 lanes that share a 128-block), and y is never rounded to 16 bits on the
// way to 8.  Bound: HBM (with a residual 7.03 bytes per element), launch latency for decode's few rows.
#include <cstdio>

#include "tg_decoder_common.cuh"

namespace tg {
namespace {

struct NormParams {
  const void* x;
  const void* residual;  // null: h = x and nothing is written to h_out
  const void* weight;
  void* h_out;
  uint8_t* y;
  float* s;
  int64_t x_pitch, r_pitch;  // elements
  int32_t chunks;            // hidden / 8
  float eps, offset, inv_hidden;
};

template <typename T>
__device__ __forceinline__ float2 weight_pair(const void* w, int i, bool f32) {
  if (f32) return __ldg(reinterpret_cast<const float2*>(w) + i);
  return unpack_pair<T>(__ldg(reinterpret_cast<const uint32_t*>(w) + i));
}

// N chunks of 8 elements per thread: chunk i * blockDim + threadIdx, so 16 neighbouring lanes hold one 128-block.
template <typename T, int N, bool kWeightF32>
__global__ void __launch_bounds__(1024) tg_rms_norm_quant_kernel(const NormParams p) {
  __shared__ float partial[32];
  const int64_t row = blockIdx.x;
  griddep_wait();
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + row * p.x_pitch);
  uint4 h[N];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = i * blockDim.x + threadIdx.x;
    h[i] = c < p.chunks ? __ldcs(x + c) : make_uint4(0, 0, 0, 0);
  }
  if (p.residual != nullptr) {
    const uint4* r = reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) + row * p.r_pitch);
    uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.h_out)) + row * p.chunks;
    uint4 rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * blockDim.x + threadIdx.x;
      rv[i] = c < p.chunks ? __ldcs(r + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * blockDim.x + threadIdx.x;
      uint32_t* a = reinterpret_cast<uint32_t*>(&h[i]);
      const uint32_t* b = reinterpret_cast<const uint32_t*>(&rv[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = unpack_pair<T>(a[j]), v = unpack_pair<T>(b[j]);
        a[j] = pack_pair<T>(u.x + v.x, u.y + v.y);
      }
      if (c < p.chunks) __stcs(out + c, h[i]);
    }
  }
  griddep_launch_dependents();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t* a = reinterpret_cast<const uint32_t*>(&h[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 u = unpack_pair<T>(a[j]);
      sum = fmaf(u.x, u.x, sum);
      sum = fmaf(u.y, u.y, sum);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = (threadIdx.x & 31) < (blockDim.x >> 5) ? partial[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const float rstd = 1.0f / sqrtf(fmaf(sum, p.inv_hidden, p.eps));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = i * blockDim.x + threadIdx.x;
    const bool live = c < p.chunks;
    const uint32_t* a = reinterpret_cast<const uint32_t*>(&h[i]);
    float y[8], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 u = unpack_pair<T>(a[j]);
      const float2 w = live ? weight_pair<T>(p.weight, c * 4 + j, kWeightF32) : make_float2(0.f, 0.f);
      y[2 * j] = u.x * rstd * (w.x + p.offset);
      y[2 * j + 1] = u.y * rstd * (w.y + p.offset);
      amax = fmaxf(amax, fmaxf(fabsf(y[2 * j]), fabsf(y[2 * j + 1])));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float scale = __fdiv_rn(amax, 448.f);
    if (scale == 0.f) scale = 1.f;
    // y is a 32-bit value of its own, so the quotient needs no correctly rounded division: y * RN(1 / s) is within 2^-23
    const bool tame = q8_scale_is_tame(scale);
    const float r = __frcp_rn(scale);
    uint32_t q[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = tame ? y[j] * r : __fdiv_rn(y[j], scale);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      q[j] = q8_cast2<kQ8E4M3>(y[4 * j], y[4 * j + 1], 0.f, 0.f) | (q8_cast2<kQ8E4M3>(y[4 * j + 2], y[4 * j + 3], 0.f, 0.f) << 16);
    if (live) {
      __stcs(reinterpret_cast<uint2*>(p.y) + row * p.chunks + c, make_uint2(q[0], q[1]));
      if ((threadIdx.x & 15) == 0) p.s[row * (p.chunks >> 4) + (c >> 4)] = scale;
    }
  }
}

template <typename T, int N>
cudaError_t launch_n(const NormParams& p, int64_t rows, int threads, bool wf32, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  return wf32 ? launch_pdl(tg_rms_norm_quant_kernel<T, N, true>, grid, block, 0, st, p)
              : launch_pdl(tg_rms_norm_quant_kernel<T, N, false>, grid, block, 0, st, p);
}

template <typename T>
cudaError_t launch(const NormParams& p, int64_t rows, int num_sms, bool wf32, cudaStream_t st) {
  // Few rows: one chunk per thread, the row's latency counts (333 x 5120: 3.6 us against 3.7 with two, 4.4 with four).
  // Many rows: two, so that the reductions are shared by more elements while the SM still holds enough threads to keep
  // loads in flight (8192 x 8192 with residual, 472 MB: 78 us = 6.0 TB/s against 96 with one, 91 with four).
  const int want = rows <= 4 * num_sms ? 1 : 2;
  int n = 1;
  while (n < 8 && (n < want || (p.chunks + n - 1) / n > 1024)) n *= 2;
  const int threads = ((p.chunks + n - 1) / n + 31) / 32 * 32;
  if (n == 1) return launch_n<T, 1>(p, rows, threads, wf32, st);
  if (n == 2) return launch_n<T, 2>(p, rows, threads, wf32, st);
  if (n == 4) return launch_n<T, 4>(p, rows, threads, wf32, st);
  return launch_n<T, 8>(p, rows, threads, wf32, st);
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" TG_API int32_t tg_rms_norm_quant(const TgTensorDesc* Y, const TgTensorDesc* S, const TgTensorDesc* H,
                                            const TgTensorDesc* X, const TgTensorDesc* R, const TgTensorDesc* W, float eps,
                                            float weight_offset, int32_t device_id, uint64_t stream) {
  if (X == nullptr || W == nullptr) return api_fail(TG_ERR_NULL, "X or W descriptor is null");
  if (!is_16bit(X->dtype)) return api_fail(TG_ERR_DTYPE, "X must be bf16 or f16");
  if (X->ndim != 2) return api_fail(TG_ERR_ARGS, "X must be 2-D (flatten the leading dimensions)");
  const int64_t T = X->shape[0], hidden = X->shape[1];
  if (T < 0 || T > 0x7fffffff || hidden < 128 || hidden % 128 != 0 || hidden > 65536)
    return api_fail(TG_ERR_ARGS, "the hidden size must be a multiple of 128 from 128 to 65536");
  const int64_t ys[2] = {T, hidden}, ss[2] = {T, hidden / 128}, ws[1] = {hidden};
  int32_t rc;
  if ((rc = check_dense_nd(Y, "Y: float8_e4m3fn, contiguous, the shape of X, 16-byte aligned", TG_F8E4M3, 2, ys, 16)) != TG_OK) return rc;
  if ((rc = check_dense_nd(S, "S: f32 [rows, hidden / 128], contiguous", TG_F32, 2, ss, 4)) != TG_OK) return rc;
  if (W->dtype != X->dtype && W->dtype != TG_F32) return api_fail(TG_ERR_DTYPE, "W must have the type of X or be f32");
  if ((rc = check_dense_nd(W, "W: [hidden], contiguous, 16-byte aligned", W->dtype, 1, ws, 16)) != TG_OK) return rc;
  if ((R == nullptr) != (H == nullptr)) return api_fail(TG_ERR_NULL, "a residual and the tensor for its sum go together");
  if (R != nullptr) {
    if ((rc = check_dense_nd(H, "H: contiguous, shape and type of X, 16-byte aligned", X->dtype, 2, ys, 16)) != TG_OK) return rc;
    if (R->ndim != 2 || R->shape[0] != T || R->shape[1] != hidden) return api_fail(TG_ERR_ARGS, "the residual must have the shape of X");
    if (R->dtype != X->dtype) return api_fail(TG_ERR_DTYPE, "the residual must have the type of X");
  }
  if (!(eps >= 0.f)) return api_fail(TG_ERR_ARGS, "eps must be >= 0");
  const TgTensorDesc* in[2] = {X, R};
  for (const TgTensorDesc* t : in) {
    if (t == nullptr || T == 0) continue;
    if (t->ptr == 0) return api_fail(TG_ERR_NULL, "a data pointer is null");
    if (t->strides[1] != 1 || t->strides[0] < 0) return api_fail(TG_ERR_ARGS, "rows of X and of the residual must be dense");
    if ((t->ptr & 15u) || (T > 1 && (t->strides[0] & 7))) return api_fail(TG_ERR_ALIGN, "rows of X and of the residual need 16-byte alignment");
  }
  if (T == 0) return TG_OK;
  if (H != nullptr) {
    // H's row t may lie on row t of an input, which its block has read by then, but not on rows that others have still to read
    const uint64_t row = static_cast<uint64_t>(hidden) * 2, h_end = H->ptr + T * row;
    for (const TgTensorDesc* t : in) {
      const uint64_t end = t->ptr + static_cast<uint64_t>(T - 1) * static_cast<uint64_t>(t->strides[0]) * 2 + row;
      if (t->ptr < h_end && H->ptr < end && !(t->ptr == H->ptr && (T == 1 || t->strides[0] == hidden)))
        return api_fail(TG_ERR_ARGS, "H overlaps rows of X or of the residual: it may only take the place of dense ones");
    }
  }
  ScopedDevice guard(device_id);
  if (guard.err != cudaSuccess) {
    cudaGetLastError();
    return api_fail(TG_ERR_DEVICE, "cannot select the CUDA device");
  }
  int num_sms = 0;
  int32_t* status = nullptr;
  if ((rc = api_init_device(device_id, &num_sms, &status)) != TG_OK) return rc;
  NormParams p = {};
  p.x = reinterpret_cast<const void*>(X->ptr);
  p.residual = R ? reinterpret_cast<const void*>(R->ptr) : nullptr;
  p.weight = reinterpret_cast<const void*>(W->ptr);
  p.h_out = H ? reinterpret_cast<void*>(H->ptr) : nullptr;
  p.y = reinterpret_cast<uint8_t*>(Y->ptr);
  p.s = reinterpret_cast<float*>(S->ptr);
  p.x_pitch = X->strides[0];
  p.r_pitch = R ? R->strides[0] : 0;
  p.chunks = static_cast<int32_t>(hidden / 8);
  p.eps = eps;
  p.offset = weight_offset;
  p.inv_hidden = 1.0f / static_cast<float>(hidden);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = X->dtype == TG_BF16 ? launch<__nv_bfloat16>(p, T, num_sms, W->dtype == TG_F32, st)
                                            : launch<__half>(p, T, num_sms, W->dtype == TG_F32, st);
  if (e != cudaSuccess) {
    char msg[160];
    snprintf(msg, sizeof(msg), "rms_norm_quant launch failed: %s", cudaGetErrorString(e));
    return api_fail(TG_ERR_LAUNCH, msg);
  }
  return TG_OK;
}
