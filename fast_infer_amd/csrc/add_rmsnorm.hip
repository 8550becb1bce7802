// The residual stream's step between two blocks of a layer, for gfx950:
//
//   h   = fp16(x + residual)                                  (one rounding, as an fp16 addition)
//   out = fp16((h * r) * weight),  r = rsqrt(sum(h^2) / hidden + eps), in fp32 from the rounded h
//
// i.e. an addition followed by rms_norm, in one pass: each element of x and residual is read
// once, h and out are written once (8 bytes an element; the two calls move 10).  Bound by
// memory (16384 x 5120, 671 MB: 104 to 108 us, 6.2 to 6.4 TB/s), and by latency for few rows (1 x 4096 1.8 us, 777 x
// 2560 4.5 us from the cache).  A row is held in registers between the sum of squares
// and the scaling; rows of more than kMaxHeld elements are read back from h.
#include <algorithm>

#include "common.h"

namespace fi {
namespace addnorm {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kMaxParts = 4;                       // 16-byte pieces a thread holds
constexpr int kMaxHeld = kThreads * 8 * kMaxParts;  // 8192
// Rows up to this wide by a wave each, wider ones by a workgroup: 60000 x 256 56 -> 22 us, 16384 x 768
// 20 -> 18, 30000 x 1024 40 -> 38.
constexpr int kNarrow = 1024;
// Bytes moved from which the non-temporal policy pays, beyond the last-level cache: 16384 x 5120
// 116 -> 110 us a call; 30000 x 1024 (246 MB) 40 against 42.
constexpr int64_t kCached = (int64_t)400 << 20;

struct Params {
  const half_t* x;
  const half_t* res;
  const half_t* weight;
  half_t* h;
  half_t* out;
  int64_t x_stride, res_stride, h_stride, out_stride;
  int64_t rows;
  int hidden;
  float eps;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

__device__ __forceinline__ u32x4 add8(u32x4 a, u32x4 b) {
  const half8 x = as_half8(a), y = as_half8(b);
  half8 s;
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = (half_t)((float)x[e] + (float)y[e]);
  return as_u32x4(s);
}

__device__ __forceinline__ float sum_sq8(u32x4 v) {
  const half8 h = as_half8(v);
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)h[e], (float)h[e], s);
  return s;
}

// fp16((h * r) * w), the products rounded separately
__device__ __forceinline__ u32x4 scale8(u32x4 hv, float r, u32x4 wv) {
#pragma clang fp contract(off)
  const half8 h = as_half8(hv), w = as_half8(wv);
  half8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (half_t)(((float)h[e] * r) * (float)w[e]);
  return as_u32x4(y);
}

// Descriptor over one row: elements past `hidden` read zeros and are not written.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const half_t* row, int hidden) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)row, (short)0, hidden * 2, 0x00020000);
}
// kNt: the non-temporal policy (2), for calls beyond the last-level cache.
template <bool kNt>
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, int byte) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, byte, 0, kNt ? 2 : 0));
}
template <bool kNt>
__device__ __forceinline__ void store16(__amdgpu_buffer_rsrc_t r, int byte, u32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(v, r, byte, 0, kNt ? 2 : 0);
}

// A row by kRowWaves waves (1 or all), kParts pieces a thread.  (Workgroups that loop over rows and
// load the next one ahead were slower: 16384 x 5120 117 to 122 us against 110.)
template <int kRowWaves, int kParts, bool kNt>
__global__ __launch_bounds__(kThreads) void held_kernel(Params p) {
  static_assert(kRowWaves == 1 || kRowWaves == kWaves, "a workgroup's waves share a row, or none do");
  __shared__ float part[kWaves];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * (kWaves / kRowWaves) + w / kRowWaves;
  if (kRowWaves < kWaves && row >= p.rows) return;
  const int at = ((w % kRowWaves) * 64 + lane) * 16;  // byte of the first piece
  constexpr int kStep = kRowWaves * 64 * 16;
  const __amdgpu_buffer_rsrc_t xr = row_rsrc(p.x + row * p.x_stride, p.hidden);
  const __amdgpu_buffer_rsrc_t rr = row_rsrc(p.res + row * p.res_stride, p.hidden);
  const __amdgpu_buffer_rsrc_t wr = row_rsrc(p.weight, p.hidden);
  u32x4 v[kParts], a[kParts], wv[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    v[i] = load16<kNt>(xr, at + i * kStep);
    a[i] = load16<kNt>(rr, at + i * kStep);
  }
#pragma unroll
  for (int i = 0; i < kParts; ++i) wv[i] = load16<false>(wr, at + i * kStep);
  const __amdgpu_buffer_rsrc_t hr = row_rsrc(p.h + row * p.h_stride, p.hidden);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    v[i] = add8(v[i], a[i]);
    store16<kNt>(hr, at + i * kStep, v[i]);
    s += sum_sq8(v[i]);
  }
  s = wave_sum(s);
  if (kRowWaves > 1) {
    if (lane == 0) part[w] = s;
    __syncthreads();
    s = part[0] + part[1] + part[2] + part[3];
  }
  const float r = rsqrtf(s / (float)p.hidden + p.eps);
  const __amdgpu_buffer_rsrc_t orr = row_rsrc(p.out + row * p.out_stride, p.hidden);
#pragma unroll
  for (int i = 0; i < kParts; ++i) store16<kNt>(orr, at + i * kStep, scale8(v[i], r, wv[i]));
}

// Rows of any length: h is read back (by the thread that wrote it).
__global__ __launch_bounds__(kThreads) void long_kernel(Params p) {
  __shared__ float part[kWaves];
  const int64_t row = blockIdx.x;
  const half_t* x = p.x + row * p.x_stride;
  const half_t* a = p.res + row * p.res_stride;
  half_t* h = p.h + row * p.h_stride;
  half_t* o = p.out + row * p.out_stride;
  float s = 0.f;
  for (int k = threadIdx.x * 8; k < p.hidden; k += kThreads * 8) {
    const u32x4 v = add8(*(const u32x4*)(x + k), *(const u32x4*)(a + k));
    *(u32x4*)(h + k) = v;
    s += sum_sq8(v);
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  const float r = rsqrtf((part[0] + part[1] + part[2] + part[3]) / (float)p.hidden + p.eps);
  for (int k = threadIdx.x * 8; k < p.hidden; k += kThreads * 8)
    *(u32x4*)(o + k) = scale8(*(const u32x4*)(h + k), r, *(const u32x4*)(p.weight + k));
}

}  // namespace addnorm
}  // namespace fi

extern "C" int fi_add_rmsnorm(const void* x, int64_t x_stride, const void* residual, int64_t res_stride,
                              int64_t M, int64_t hidden, const void* weight, float eps, void* h_out,
                              int64_t h_stride, void* out, int64_t out_stride, void* stream) {
  using namespace fi;
  using namespace fi::addnorm;
  static const char* fn = "fi_add_rmsnorm";
  clear_error();
  if (M < 0 || hidden <= 0 || hidden % 8 != 0 || hidden > (1 << 24)) {
    set_error("%s: %lld rows of %lld elements not supported (hidden a multiple of 8 up to 2^24)", fn,
              (long long)M, (long long)hidden);
    return FI_ERR_UNSUPPORTED;
  }
  if (M == 0) return FI_OK;
  if (!x || !residual || !weight || !h_out || !out) {
    set_error("%s: null pointer", fn);
    return FI_ERR_INVALID;
  }
  if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)h_out | (uintptr_t)out) & 15u) ||
      (x_stride | res_stride | h_stride | out_stride) % 8 != 0) {
    set_error("%s: rows must be 16-byte aligned (strides multiple of 8)", fn);
    return FI_ERR_INVALID;
  }
  if (h_out == out || (M > 1 && (h_stride < hidden || out_stride < hidden))) {
    set_error("%s: h_out and out must not overlap, nor the rows of either", fn);
    return FI_ERR_INVALID;
  }
  if (M >= (1 << 24)) {  // 256 threads a row: a launch takes fewer than 2^32
    set_error("%s: too many rows (%lld)", fn, (long long)M);
    return FI_ERR_UNSUPPORTED;
  }
  const Params p = {(const half_t*)x, (const half_t*)residual, (const half_t*)weight, (half_t*)h_out,
                    (half_t*)out, x_stride, res_stride, h_stride, out_stride, M, (int)hidden, eps};
  const hipStream_t st = (hipStream_t)stream;
  const dim3 block(kThreads);
  if (hidden > kMaxHeld) {
    hipLaunchKernelGGL(long_kernel, dim3((unsigned)M), block, 0, st, p);
    return check_launch(fn);
  }
  const bool nt = M * hidden * 8 > kCached;
  const bool narrow = hidden <= kNarrow;
  const int64_t wgs = narrow ? (M + kWaves - 1) / kWaves : M;
  const dim3 grid((unsigned)wgs);
  const int parts = (int)((hidden + (narrow ? 512 : 2048) - 1) / (narrow ? 512 : 2048));
#define FI_ADDNORM(R, P)                                                              \
  do {                                                                                \
    if (nt)                                                                           \
      hipLaunchKernelGGL((held_kernel<R, P, true>), grid, block, 0, st, p);           \
    else                                                                              \
      hipLaunchKernelGGL((held_kernel<R, P, false>), grid, block, 0, st, p);          \
  } while (0)
  switch (narrow ? -parts : parts) {
    case -1: FI_ADDNORM(1, 1); break;
    case -2: FI_ADDNORM(1, 2); break;
    case 1: FI_ADDNORM(4, 1); break;
    case 2: FI_ADDNORM(4, 2); break;
    case 3: FI_ADDNORM(4, 3); break;
    default: FI_ADDNORM(4, 4); break;
  }
#undef FI_ADDNORM
  return check_launch(fn);
}
