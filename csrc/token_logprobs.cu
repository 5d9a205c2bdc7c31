// Log-probability of a given token, entropy and the most likely tokens of each
// row of logits, in one pass over the row.
//
//   m = max x,  Z = sum e^(x - m),  S = sum e^(x - m) (x - m)
//   logprob = x[id] - m - log Z,    entropy = log Z - S / Z
//
// A term with e^(x - m) = 0 adds nothing to S (x = -inf included). A row
// without a finite maximum (all -inf, a +inf or a NaN) has no distribution:
// its log-probabilities and entropy are NaN. In the order of the top tokens a
// NaN counts as larger than every number; equal logits go by index.
//
// What bounds it is reading the logits once. A warp takes blocks of 512
// elements, the next block on its way while one is summed: the block's maximum
// by one warp reduction (a running maximum of the warp's, so that sums are
// rescaled only when it moves), then an exponential and four adds and multiplies
// per element, in pairs. x - m comes before the factor log2(e): a mask of the
// type's lowest value would leave fp32's range with it.
//
// The top tokens cost the pass nothing but the block maxima, which it has
// anyway and leaves behind: the k blocks with the largest maxima (the earlier
// one of equals) hold the k largest elements, since each block left out has k
// elements before it in the order. After the pass one CTA per row picks those
// blocks, reads them again (k KB, from L2) and ranks the few elements that reach
// the smallest of the picked maxima.
//
// Few rows are split over several CTAs: each leaves (m, Z, S) and its block
// maxima in the workspace, and the CTA that counts the row's last part
// finishes the row.

#include "ragged.cuh"

namespace afd {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = 512;             // elements of a block: 16 a lane
constexpr int kMaxBlocks = kMaxLogprobVocab / kBlock;
constexpr int kList = 2048;             // elements above the threshold at most (see refine)
constexpr int kTies = 256;              // elements at the threshold kept before k are picked in order
constexpr float kLog2e = 1.4426950408889634f;

// Floats in an order that unsigned integers have, NaN last; never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ float max3n(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float d;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

// A lane's 16 elements of a block: two runs of 8 neighbours, 256 elements apart,
// where rows are 16-byte aligned (kVec); every 32nd element elsewhere.
template <typename T, bool kVec>
struct Lane {
  static constexpr int kWords = 16 * sizeof(T) / 4;
  uint32_t w[kWords];

  static __device__ __forceinline__ int index(int lane, int e) {
    return kVec ? (e / 8) * 256 + lane * 8 + e % 8 : e * 32 + lane;
  }
  __device__ __forceinline__ void set(int e, float v) {
    if constexpr (sizeof(T) == 4) {
      w[e] = __float_as_uint(v);
    } else {
      const T t = from_f<T>(v);
      const uint32_t b = *reinterpret_cast<const uint16_t*>(&t);
      w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | (b << 16) : (w[e / 2] & 0xffff0000u) | b;
    }
  }
  // Elements of the block at x[at ..]; -inf past the row's end.
  __device__ __forceinline__ void load(const T* x, int at, int V, int lane) {
    if (kVec && at + kBlock <= V) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < kWords / 8; ++q) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + at + h * 256 + lane * 8) + q);
          const int o = h * (kWords / 2) + q * 4;
          w[o] = v.x;
          w[o + 1] = v.y;
          w[o + 2] = v.z;
          w[o + 3] = v.w;
        }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = at + index(lane, e);
        if constexpr (sizeof(T) == 4) {
          w[e] = i < V ? __float_as_uint(x[i]) : 0xff800000u;
        } else {
          set(e, i < V ? to_f(x[i]) : -INFINITY);
        }
      }
    }
  }
  __device__ __forceinline__ float2 pair(int p) const {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(w[2 * p]), __uint_as_float(w[2 * p + 1]));
    else
      return unpack2<T>(w[p]);
  }
};

// e^d for d <= 0; from kGone down it is 0, and so is e^d d.
constexpr float kGone = -1000.f;
__device__ __forceinline__ float exp_neg(float d) { return exp2_approx(d * kLog2e); }

// (m, Z, S) of some elements; m = +inf stands for a NaN too.
struct Sums {
  float m, z, s;
};

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, 0.f, 0.f};
  const float da = fmaxf(a.m - m, kGone), db = fmaxf(b.m - m, kGone);
  const float ca = exp_neg(da), cb = exp_neg(db);
  return {m, a.z * ca + b.z * cb, ca * (a.s + a.z * da) + cb * (b.s + b.z * db)};
}

struct Shared {
  Sums sums[kWarps];
  int sel[kMaxTopLogprobs];
  uint32_t thr;
  int n_sel, n_list, n_ties, last;
  uint32_t most[kThreads];
  unsigned long long list[kList + kTies];
  uint32_t keys[1];  // [blocks], of the dynamic part
};

// The top_k elements of row x as (key, ~index) in sh.list, unsorted, from the
// block maxima in sh.keys; returns how many were listed (top_k at least).
template <typename T, bool kVec>
__device__ int list_top(Shared& sh, const T* x, int V, int n_blocks, int top_k) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (warp == 0) {
    // top_k rounds: the largest key left, the first block of equals
    const int n = min(top_k, n_blocks);
    uint32_t best = 0;
    int at = 0;
    auto look = [&]() {
      best = 0;
      for (int i = lane; i < n_blocks; i += 32)
        if (sh.keys[i] > best) {
          best = sh.keys[i];
          at = i;
        }
    };
    look();
    uint32_t k = 0;
    for (int r = 0; r < n; ++r) {
      k = __reduce_max_sync(0xffffffffu, best);
      const int b = (int)__reduce_min_sync(0xffffffffu, best == k ? (unsigned)at : 0xffffffffu);
      if (lane == 0) sh.sel[r] = b;
      if (best == k && at == b) {
        sh.keys[b] = 0;
        look();
      }
      __syncwarp();
    }
    if (lane == 0) {
      sh.n_sel = n;
      sh.thr = n == top_k ? k : 0;
      sh.n_list = sh.n_ties = 0;
    }
  }
  __syncthreads();
  const int n_sel = sh.n_sel;
  // every element of the picked blocks, with its key (0 past the row's end)
  auto each = [&](auto&& f) {
    for (int b = warp; b < n_sel; b += kWarps) {
      Lane<T, kVec> v;
      const int at = sh.sel[b] * kBlock;
      v.load(x, at, V, lane);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float2 p = v.pair(e / 2);
        const int i = at + Lane<T, kVec>::index(lane, e);
        f(i < V ? order_of(e % 2 ? p.y : p.x) : 0u, i);
      }
    }
  };
  auto collect = [&]() {
    const uint32_t thr = sh.thr;
    each([&](uint32_t k, int i) {
      if (k >= thr && k != 0) {
        const bool tie = k == thr;
        const int at = atomicAdd(tie ? &sh.n_ties : &sh.n_list, 1);
        if (at < (tie ? kTies : kList))
          sh.list[tie ? kList + at : at] = ((unsigned long long)k << 32) | (uint32_t)~i;
      }
    });
    __syncthreads();
  };
  if (n_sel == top_k) collect();
  if (n_sel < top_k || sh.n_list > kList) {
    // A nearer threshold: the top_k-th of the threads' largest keys. At most
    // top_k - 1 <= 31 threads hold elements above it, of the 64 at most that a
    // thread sees: they fit the list.
    uint32_t mine = 0;
    each([&](uint32_t k, int) { mine = max(mine, k); });
    sh.most[threadIdx.x] = mine;
    __syncthreads();
    int rank = 0;
    for (int t = 0; t < kThreads; ++t) {
      const uint32_t k = sh.most[t];
      rank += k > mine || (k == mine && t < (int)threadIdx.x);
    }
    if (rank == top_k - 1) sh.thr = mine;
    if (threadIdx.x == 0) sh.n_list = sh.n_ties = 0;
    __syncthreads();
    collect();
  }
  if (sh.n_ties > kTies) {
    // more equal elements than the list takes: the first ones by index, block
    // by block (the first blocks hold enough of them, or few blocks do)
    __syncthreads();
    if (warp == 0) {
      const uint32_t thr = sh.thr;
      const int mine = lane < n_sel ? sh.sel[lane] : 0x7fffffff;
      int n = 0;
      for (int last = -1, b = 0; b < n_sel && n < top_k; ++b) {
        last = (int)__reduce_min_sync(0xffffffffu, mine > last ? (unsigned)mine : 0x7fffffffu);
        for (int c = 0; c < kBlock && n < top_k; c += 32) {
          const int i = last * kBlock + c + lane;
          const bool tie = i < V && order_of(to_f(x[i])) == thr;
          const unsigned set = __ballot_sync(0xffffffffu, tie);
          const int at = n + __popc(set & ((1u << lane) - 1));
          if (tie && at < kTies)
            sh.list[kList + at] = ((unsigned long long)thr << 32) | (uint32_t)~i;
          n += __popc(set);
        }
      }
      __syncwarp();
      if (lane == 0) sh.n_ties = min(n, kTies);
    }
    __syncthreads();
  }
  // one list
  const int n = sh.n_list, ties = sh.n_ties;
  unsigned long long t = 0;
  if ((int)threadIdx.x < ties) t = sh.list[kList + threadIdx.x];
  __syncthreads();
  if ((int)threadIdx.x < ties) sh.list[n + threadIdx.x] = t;
  __syncthreads();
  return n + ties;
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads, 4)
    token_logprobs_kernel(TokenLogprobsArgs a, int splits, int n_blocks) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int r = blockIdx.x / splits, split = blockIdx.x % splits;
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)r * a.row;
  const int first = (int)((long long)n_blocks * split / splits);
  const int end = (int)((long long)n_blocks * (split + 1) / splits);
  uint32_t* keys = splits > 1 ? a.block_keys + (size_t)r * n_blocks : sh.keys;

  float m = -INFINITY;  // of this warp's blocks
  float2 z2 = make_float2(0.f, 0.f), s2 = make_float2(0.f, 0.f);
  Lane<T, kVec> cur, next;
  int b = first + warp;
  if (b < end) cur.load(x, b * kBlock, a.V, lane);
  for (; b < end; b += kWarps) {
    if (b + kWarps < end) next.load(x, (b + kWarps) * kBlock, a.V, lane);
    float2 v[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) v[p] = cur.pair(p);
    float mx = max3n(v[0].x, v[0].y, v[1].x);
    float my = max3n(v[1].y, v[2].x, v[2].y);
#pragma unroll
    for (int p = 3; p < 7; p += 2) {
      mx = max3n(mx, v[p].x, v[p].y);
      my = max3n(my, v[p + 1].x, v[p + 1].y);
    }
    mx = warp_max_nan(max3n(max3n(mx, v[7].x, v[7].y), my, my));
    if (a.top_k > 0 && lane == 0) keys[b] = order_of(mx);
    if (mx != mx) m = INFINITY;
    if (mx > -INFINITY && m < INFINITY) {
      if (mx > m) {
        const float d = fmaxf(m - mx, kGone), c = exp_neg(d);
        s2 = make_float2((s2.x + z2.x * d) * c, (s2.y + z2.y * d) * c);
        z2 = make_float2(z2.x * c, z2.y * c);
        m = mx;
      }
      const float2 nm = make_float2(-m, -m), l2 = make_float2(kLog2e, kLog2e);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        float2 d = add2(v[p], nm);
        d.x = fmaxf(d.x, kGone);
        d.y = fmaxf(d.y, kGone);
        const float2 t = mul2(d, l2);
        const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
        z2 = add2(z2, e);
        s2 = fma2(e, d, s2);
      }
    }
    cur = next;
  }
  Sums mine = {m, z2.x + z2.y, s2.x + s2.y};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {  // one m for the whole warp
    mine.z += __shfl_xor_sync(0xffffffffu, mine.z, o);
    mine.s += __shfl_xor_sync(0xffffffffu, mine.s, o);
  }
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  Sums all = sh.sums[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) all = join(all, sh.sums[w]);
  if (splits > 1) {
    float* part = a.parts + ((size_t)r * splits + split) * 4;
    if (threadIdx.x == 0)
      *reinterpret_cast<float4*>(part) = make_float4(all.m, all.z, all.s, 0.f);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      sh.last = atomicAdd(&a.counters[r], 1) == splits - 1;
      if (sh.last) a.counters[r] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    if (a.top_k > 0)
      for (int i = threadIdx.x; i < n_blocks; i += kThreads) sh.keys[i] = __ldcg(keys + i);
    all = {-INFINITY, 0.f, 0.f};
    for (int i = lane; i < splits; i += 32) {
      const float4 p = __ldcg(reinterpret_cast<const float4*>(a.parts) + (size_t)r * splits + i);
      all = join(all, {p.x, p.y, p.z});
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Sums other = {__shfl_xor_sync(0xffffffffu, all.m, o),
                          __shfl_xor_sync(0xffffffffu, all.z, o),
                          __shfl_xor_sync(0xffffffffu, all.s, o)};
      // the same order on both sides of the exchange
      all = lane & o ? join(other, all) : join(all, other);
    }
    __syncthreads();
  }
  const bool none = !(all.m > -INFINITY && all.m < INFINITY);
  const float lz = logf(all.z);
  auto logprob = [&](float v) { return none ? NAN : v - all.m - lz; };
  if (threadIdx.x == 0) {
    const int64_t id = a.ids[r];
    a.logprob[r] = id >= 0 && id < a.V ? logprob(to_f(x[id])) : NAN;
    a.entropy[r] = none ? NAN : lz - all.s / all.z;
  }
  if (a.top_k == 0) return;
  const int n = list_top<T, kVec>(sh, x, a.V, n_blocks, a.top_k);
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const unsigned long long k = sh.list[c];
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += sh.list[o] > k;
    if (rank < a.top_k) {
      a.top_ids[(size_t)r * a.top_k + rank] = (int64_t)(uint32_t)~(uint32_t)k;
      a.top_logprobs[(size_t)r * a.top_k + rank] = logprob(value_of((uint32_t)(k >> 32)));
    }
  }
}

template <typename T>
int launch_one(const TokenLogprobsArgs& a, int splits, int n_blocks, cudaStream_t s) {
  const size_t bytes = sizeof(Shared) + (size_t)(a.top_k > 0 ? n_blocks : 0) * 4;
  const bool vec = ((uintptr_t)a.logits & 15) == 0 &&
                   (a.R == 1 || a.row * (long long)sizeof(T) % 16 == 0);
  const auto kern = vec ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern),
                                       (int)(sizeof(Shared) + kMaxBlocks * 4));
  if (e == cudaSuccess)
    e = launch_k(kern, dim3((unsigned)(a.R * splits)), dim3(kThreads), bytes, s, a, splits,
                 n_blocks);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

int blocks_of(int V) { return (V + kBlock - 1) / kBlock; }

}  // namespace

// CTAs of a row: enough for six on each SM in all, a block for each warp at least.
int token_logprobs_splits(int R, int V, int num_sms) {
  const int most = (blocks_of(V) + kWarps - 1) / kWarps;
  const long long want = R > 0 ? (6ll * num_sms + R - 1) / R : 1;
  return (int)(want < most ? want : most);
}

long long token_logprobs_workspace(int R, int V, int splits) {
  return splits > 1 ? (long long)R * (16ll * splits + 4ll * blocks_of(V)) : 0;
}

int launch_token_logprobs(const TokenLogprobsArgs& a_in, int splits, void* ws, cudaStream_t s) {
  TokenLogprobsArgs a = a_in;
  if (a.R == 0) return 0;
  if (a.V > kMaxLogprobVocab || (long long)a.R * splits > 0x7fffffff) return 1;
  const int n_blocks = blocks_of(a.V);
  a.parts = reinterpret_cast<float*>(ws);
  a.block_keys = reinterpret_cast<uint32_t*>(a.parts + (size_t)a.R * splits * 4);
  if (a.elem == kElemBf16) return launch_one<__nv_bfloat16>(a, splits, n_blocks, s);
  if (a.elem == kElemF16) return launch_one<__half>(a, splits, n_blocks, s);
  return launch_one<float>(a, splits, n_blocks, s);
}

}  // namespace afd
