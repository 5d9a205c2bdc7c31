// Attention of one new token per sequence over the paged KV cache.
//
// out[b, h] = sum_j p_j v_j, p = softmax over j < seq_lens[b] of
// q[b, h] . k_j * scale, with h's kv head h / (nq / nkv).

#include "ragged.cuh"

namespace afd {

namespace {

// One CTA of 8 warps per (sequence, head): the warps take every eighth key,
// each with its own running maximum and sum, and join at the end.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_decode_kernel(PagedDecodeArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  __shared__ float om[8][D], mm[8], ll[8];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int b = blockIdx.x / a.nq, h = blockIdx.x % a.nq, kvh = h / (a.nq / a.nkv);
  const T* q = reinterpret_cast<const T*>(a.q) + (size_t)b * a.q_row + (size_t)h * D;
  const int len = checked_len(a.seq_lens[b], a.max_pages * a.page_size, a.status, 221);
  float qv[E], o[E];
  for (int i = 0; i < E; ++i) {
    qv[i] = to_f(q[lane * E + i]) * a.scale;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = warp; j < len; j += 8) {
    const int page = a.page_table[(size_t)b * a.table_row + j / a.page_size];
    const bool ok = page >= 0 && page < a.num_pages;
    if (!ok) report_status(a.status, kBoundsViolation, 222);
    const size_t at = (size_t)(ok ? page : 0) * a.page_stride +
                      ((size_t)kvh * a.page_size + j % a.page_size) * D;
    const T* k = reinterpret_cast<const T*>(a.k_pages) + at;
    const T* v = reinterpret_cast<const T*>(a.v_pages) + at;
    float s = 0.f;
    for (int i = 0; i < E; ++i) s += qv[i] * (ok ? to_f(k[lane * E + i]) : 0.f);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float m_new = fmaxf(m, s);
    const float c = m_new == -INFINITY ? 1.f : __expf(m - m_new);
    const float p = m_new == -INFINITY ? 0.f : __expf(s - m_new);
    l = l * c + p;
    for (int i = 0; i < E; ++i) o[i] = o[i] * c + p * (ok ? to_f(v[lane * E + i]) : 0.f);
    m = m_new;
  }
  for (int i = 0; i < E; ++i) om[warp][lane * E + i] = o[i];
  if (lane == 0) {
    mm[warp] = m;
    ll[warp] = l;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int w = 0; w < 8; ++w) M = fmaxf(M, mm[w]);
    for (int w = 0; w < 8; ++w) {
      const float c = mm[w] == -INFINITY ? 0.f : __expf(mm[w] - M);
      L += ll[w] * c;
      acc += om[w][threadIdx.x] * c;
    }
    T* out = reinterpret_cast<T*>(a.out) + ((size_t)b * a.nq + h) * D;
    out[threadIdx.x] = from_f<T>(L > 0.f ? acc / L : 0.f);
  }
}

}  // namespace

int launch_paged_decode(const PagedDecodeArgs& a, cudaStream_t s) {
  if (a.B == 0) return 0;
  const dim3 grid((unsigned)(a.B * a.nq));
  cudaError_t e;
  if (a.elem == kElemBf16)
    e = a.D == 128 ? launch_k(paged_decode_kernel<__nv_bfloat16, 128>, grid, dim3(256), 0, s, a)
                   : launch_k(paged_decode_kernel<__nv_bfloat16, 64>, grid, dim3(256), 0, s, a);
  else
    e = a.D == 128 ? launch_k(paged_decode_kernel<__half, 128>, grid, dim3(256), 0, s, a)
                   : launch_k(paged_decode_kernel<__half, 64>, grid, dim3(256), 0, s, a);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

}  // namespace afd
