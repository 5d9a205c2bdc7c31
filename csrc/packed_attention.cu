// Causal attention of packed queries over packed keys or over the paged cache.
//
// out[r, h] = sum_j p_j v_j,  p = softmax over the visible keys j <= pos(r) of
// q[r, h] . k_j * scale, with h's kv head h / (nq / nkv).

#include "ragged.cuh"

namespace afd {

namespace {

// One warp per (query row, head); the lanes split the head dim, and each key
// updates the running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(128) packed_attention_kernel(PackedAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32;
  const long long gw = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  if (gw >= (long long)a.T * a.nq) return;
  const int row = (int)(gw / a.nq), h = (int)(gw % a.nq), kvh = h / (a.nq / a.nkv);
  constexpr int E = D / 32;
  const T* q = reinterpret_cast<const T*>(a.q) + (size_t)row * a.q_row + (size_t)h * D;
  float qv[E], o[E];
  for (int i = 0; i < E; ++i) {
    qv[i] = to_f(q[lane * E + i]) * a.scale;
    o[i] = 0.f;
  }
  // the last sequence that starts at or before this row
  int lo = 0, hi = a.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.cu_q[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int q0 = a.cu_q[lo], q1 = min(a.cu_q[lo + 1], a.T);
  int len = 0, k0 = 0;
  if (a.n_seqs > 0 && row >= q0 && row < q1) {
    if (a.paged) {
      len = checked_len(a.seq_lens[lo], a.max_pages * a.page_size, a.status, 211);
    } else {
      k0 = min(max(a.cu_k[lo], 0), a.Tk);
      len = min(max(a.cu_k[lo + 1], k0), a.Tk) - k0;
      if (k0 != a.cu_k[lo] || k0 + len != a.cu_k[lo + 1])
        report_status(a.status, kBoundsViolation, 212);
    }
  }
  const int pos = len > 0 ? len - (q1 - row) : -1;
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j <= pos; ++j) {
    const T *k, *v;
    bool ok = true;
    if (a.paged) {
      const int page = a.page_table[(size_t)lo * a.table_row + j / a.page_size];
      ok = page >= 0 && page < a.num_pages;
      const size_t at = (size_t)(ok ? page : 0) * a.page_stride +
                        ((size_t)kvh * a.page_size + j % a.page_size) * D;
      k = reinterpret_cast<const T*>(a.k_pages) + at;
      v = reinterpret_cast<const T*>(a.v_pages) + at;
      if (!ok) report_status(a.status, kBoundsViolation, 213);
    } else {
      k = reinterpret_cast<const T*>(a.k) + (size_t)(k0 + j) * a.k_row + (size_t)kvh * D;
      v = reinterpret_cast<const T*>(a.v) + (size_t)(k0 + j) * a.v_row + (size_t)kvh * D;
    }
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
  T* out = reinterpret_cast<T*>(a.out) + ((size_t)row * a.nq + h) * D;
  for (int i = 0; i < E; ++i) out[lane * E + i] = from_f<T>(l > 0.f ? o[i] / l : 0.f);
}

}  // namespace

int launch_packed_attention(const PackedAttnArgs& a, cudaStream_t s) {
  if (a.T == 0) return 0;
  const dim3 grid((unsigned)(((long long)a.T * a.nq + 3) / 4));
  cudaError_t e;
  if (a.elem == kElemBf16)
    e = a.D == 128 ? launch_k(packed_attention_kernel<__nv_bfloat16, 128>, grid, dim3(128), 0, s, a)
                   : launch_k(packed_attention_kernel<__nv_bfloat16, 64>, grid, dim3(128), 0, s, a);
  else
    e = a.D == 128 ? launch_k(packed_attention_kernel<__half, 128>, grid, dim3(128), 0, s, a)
                   : launch_k(packed_attention_kernel<__half, 64>, grid, dim3(128), 0, s, a);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

}  // namespace afd
