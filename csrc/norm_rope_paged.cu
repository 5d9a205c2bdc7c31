// Per-head RMSNorm and RoPE of the q and k heads of a packed qkv projection,
// with k and v stored into the pages of the KV cache (or k packed).
//
//   y = x / sqrt(mean(x^2) + eps) * w,   out[j]       = y[j] cos - y[j + D/2] sin
//                                        out[j + D/2] = y[j + D/2] cos + y[j] sin
//
// Everything between the load and the store is fp32 with one rounding at the
// store. The model's padded path rounds after the norm, the weight and each
// RoPE product, as HF's eager code does; here a single rounding is both
// closer to the formula and cheaper.

#include "ragged.cuh"

namespace afd {

namespace {

template <typename T>
__global__ void __launch_bounds__(256) norm_rope_kernel(NormRopeArgs a) {
  pdl_wait();
  pdl_trigger();
  const int heads = a.nq + 2 * a.nkv;
  const long long gw = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (gw >= (long long)a.T * heads) return;
  const int t = (int)(gw / heads), h = (int)(gw % heads);
  const int D = a.D, half = D / 2, per = half / 32;  // 1 or 2 pairs a lane
  const T* src = reinterpret_cast<const T*>(a.qkv) + (size_t)t * a.qkv_row + (size_t)h * D;

  T* dst = nullptr;
  if (h < a.nq) {
    dst = reinterpret_cast<T*>(a.q_out) + ((size_t)t * a.nq + h) * D;
  } else {
    const bool is_k = h < a.nq + a.nkv;
    const int kvh = is_k ? h - a.nq : h - a.nq - a.nkv;
    if (a.k_pages != nullptr) {
      const int64_t slot = a.slots[t];
      if (slot < 0) return;
      if (slot >= (int64_t)a.num_pages * a.page_size) {
        if (lane == 0) report_status(a.status, kBoundsViolation, 201);
        return;
      }
      T* pool = reinterpret_cast<T*>(is_k ? a.k_pages : a.v_pages);
      dst = pool + (slot / a.page_size) * a.page_stride +
            ((size_t)kvh * a.page_size + slot % a.page_size) * D;
    } else {
      if (!is_k) return;
      dst = reinterpret_cast<T*>(a.k_out) + ((size_t)t * a.nkv + kvh) * D;
    }
    if (!is_k) {
      for (int j = lane; j < D; j += 32) dst[j] = src[j];
      return;
    }
  }
  int pos = a.positions[t];
  if (pos < 0 || pos >= a.max_pos) {
    if (lane == 0) report_status(a.status, kBoundsViolation, 202);
    pos = min(max(pos, 0), a.max_pos - 1);
  }
  const T* w = reinterpret_cast<const T*>(h < a.nq ? a.q_norm : a.k_norm);
  float lo[2], hi[2], ss = 0.f;
  for (int i = 0; i < per; ++i) {
    lo[i] = to_f(src[lane + 32 * i]);
    hi[i] = to_f(src[half + lane + 32 * i]);
    ss += lo[i] * lo[i] + hi[i] * hi[i];
  }
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(ss / (float)D + a.eps);
  const float* cs = a.rope + (size_t)pos * D;
  for (int i = 0; i < per; ++i) {
    const int j = lane + 32 * i;
    const float x = lo[i] * r * to_f(w[j]), y = hi[i] * r * to_f(w[half + j]);
    dst[j] = from_f<T>(x * cs[j] - y * cs[half + j]);
    dst[half + j] = from_f<T>(y * cs[j] + x * cs[half + j]);
  }
}

}  // namespace

int launch_norm_rope(const NormRopeArgs& a, cudaStream_t s) {
  if (a.T == 0) return 0;
  const long long warps = (long long)a.T * (a.nq + 2 * a.nkv);
  const unsigned grid = (unsigned)((warps + 7) / 8);
  const cudaError_t e =
      a.elem == kElemBf16
          ? launch_k(norm_rope_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s, a)
          : launch_k(norm_rope_kernel<__half>, dim3(grid), dim3(256), 0, s, a);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

}  // namespace afd
