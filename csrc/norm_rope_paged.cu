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
//
// Bound by the HBM: qkv is read and q, k, v are written once. D / 16 lanes take a
// head, each with two runs of 8 elements (16 bytes) that RoPE pairs, and keep
// the loads of kHeads heads of their token on the way at once; the table's
// row and the page slot, of the token, come with them.
//
// Measured (8191 tokens, 32 + 4 heads of 128, bf16, 172 MB read and written):
// 37 us, 4.6 TB/s. One head at a time 41.6, four in blocks of 256 threads 44,
// a head a thread block with 2-byte loads 130.

#include "ragged.cuh"

namespace afd {

namespace {

constexpr int kHeads = 2;
constexpr int kThreads = 128;

template <typename T>
__device__ __forceinline__ void widen(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = unpack2<T>(w[i]);
    x[2 * i] = p.x;
    x[2 * i + 1] = p.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                    pack2<T>(x[6], x[7]));
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(NormRopeArgs a, int groups) {
  constexpr int kLanes = D / 16;  // of a head
  pdl_wait();
  pdl_trigger();
  const long long unit = ((long long)blockIdx.x * kThreads + threadIdx.x) / kLanes;
  const int sub = threadIdx.x % kLanes;
  // a unit past the end repeats the last one without storing: its warp's
  // shuffles stay whole
  const bool live = unit < (long long)a.T * groups;
  const int t = live ? (int)(unit / groups) : a.T - 1;
  const int h0 = (int)(unit % groups) * kHeads;
  const int heads = a.nq + (a.k_pages != nullptr ? 2 : 1) * a.nkv;
  const T* src = reinterpret_cast<const T*>(a.qkv) + (size_t)t * a.qkv_row + sub * 8;
  uint4 lo[kHeads], hi[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const T* x = src + (size_t)min(h0 + i, heads - 1) * D;
    lo[i] = *reinterpret_cast<const uint4*>(x);
    hi[i] = *reinterpret_cast<const uint4*>(x + D / 2);
  }
  int pos = a.positions[t];
  T *kt = nullptr, *vt = nullptr;  // the token's k and v rows of kv head 0
  int head_step = a.nkv;           // rows between kv heads
  if (a.k_pages == nullptr) {
    kt = reinterpret_cast<T*>(a.k_out) + (size_t)t * a.nkv * D;
    head_step = 1;
  } else {
    const int64_t slot = a.slots[t];
    if (slot >= (int64_t)a.num_pages * a.page_size) {
      if (live && sub == 0) report_status(a.status, kBoundsViolation, 201);
    } else if (slot >= 0) {
      const int page = (int)(slot / a.page_size), row = (int)(slot - (int64_t)page * a.page_size);
      const size_t at = (size_t)page * a.page_stride + (size_t)row * D;
      kt = reinterpret_cast<T*>(a.k_pages) + at;
      vt = reinterpret_cast<T*>(a.v_pages) + at;
    }
    head_step = a.page_size;
  }
  if (pos < 0 || pos >= a.max_pos) {
    if (live && sub == 0) report_status(a.status, kBoundsViolation, 202);
    pos = min(max(pos, 0), a.max_pos - 1);
  }
  float c[8], s[8];
  {
    const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * D + sub * 8);
    *reinterpret_cast<float4*>(c) = cs[0];
    *reinterpret_cast<float4*>(c + 4) = cs[1];
    *reinterpret_cast<float4*>(s) = cs[D / 8];
    *reinterpret_cast<float4*>(s + 4) = cs[D / 8 + 1];
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    const bool is_q = h < a.nq, is_v = h >= a.nq + a.nkv;
    T* dst = is_q ? reinterpret_cast<T*>(a.q_out) + ((size_t)t * a.nq + h) * D
             : is_v ? (vt == nullptr ? nullptr : vt + (size_t)(h - a.nq - a.nkv) * head_step * D)
                    : (kt == nullptr ? nullptr : kt + (size_t)(h - a.nq) * head_step * D);
    float x[8], y[8], ss = 0.f;
    widen<T>(lo[i], x);
    widen<T>(hi[i], y);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!live || h >= heads || dst == nullptr) continue;
    uint4 vx = lo[i], vy = hi[i];
    if (!is_v) {
      const float r = rsqrtf(ss / (float)D + a.eps);
      const T* w = reinterpret_cast<const T*>(is_q ? a.q_norm : a.k_norm) + sub * 8;
      float wx[8], wy[8];
      widen<T>(*reinterpret_cast<const uint4*>(w), wx);
      widen<T>(*reinterpret_cast<const uint4*>(w + D / 2), wy);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = x[e] * r * wx[e], v = y[e] * r * wy[e];
        x[e] = u * c[e] - v * s[e];
        y[e] = v * c[e] + u * s[e];
      }
      vx = narrow<T>(x);
      vy = narrow<T>(y);
    }
    *reinterpret_cast<uint4*>(dst + sub * 8) = vx;
    *reinterpret_cast<uint4*>(dst + D / 2 + sub * 8) = vy;
  }
}

template <typename T>
cudaError_t launch_one(const NormRopeArgs& a, cudaStream_t s) {
  const int heads = a.nq + (a.k_pages != nullptr ? 2 : 1) * a.nkv;
  const int groups = (heads + kHeads - 1) / kHeads;
  const long long lanes = (long long)a.T * groups * (a.D / 16);
  const dim3 grid((unsigned)((lanes + kThreads - 1) / kThreads));
  return a.D == 128 ? launch_k(norm_rope_kernel<T, 128>, grid, dim3(kThreads), 0, s, a, groups)
                    : launch_k(norm_rope_kernel<T, 64>, grid, dim3(kThreads), 0, s, a, groups);
}

}  // namespace

int launch_norm_rope(const NormRopeArgs& a, cudaStream_t s) {
  if (a.T == 0) return 0;
  const cudaError_t e =
      a.elem == kElemBf16 ? launch_one<__nv_bfloat16>(a, s) : launch_one<__half>(a, s);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

}  // namespace afd
