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
// rescaled only when it moves), then a subtraction, a product, an exponential, an add
// and a multiply-add per element, in pairs. A block costs about 160 instructions for 16
// exponentials a lane: 71% of the issue slots and 59% of the special function units
// are busy (1184 rows, by counter), and issue comes next after the memory.
//
// The top tokens cost the pass nothing but the block maxima, which it has
// anyway and leaves behind: the k blocks with the largest maxima (the earlier
// one of equals) hold the k largest elements, since each block left out has k
// elements before it in the order. After the pass one CTA per row picks those
// blocks, reads them again (k KB, from L2) and ranks the few elements that reach
// the smallest of the picked maxima.
//
// Measured (4096 rows of 151936, bf16, top 8; 1245 MB): 220 us in a burst, 5.7 TB/s, and
// 247 to 259 in calls repeated for half a second, at lower clocks. Earlier forms, in
// bursts: blocks loaded to registers one ahead 323, the ring with the maxima in fp32
// 250; with one multiply-add for an exponent 212, and 216 without a sum of each block (see
// Running).
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
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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

// A warp's blocks on their way, in shared memory: each lane copies what it will
// read, so no lane waits for another.
// Three deep: fp32 rows 4% faster than with four (1024 rows 99 us, 103), 33 rows 8%
// (15.5, 16.9), bf16 the same; five lose 2%.
constexpr int kStages = 3;
template <typename T>
struct Ring {
  static constexpr int kParts = sizeof(T);  // 16-byte parts of a lane
  uint4 part[kStages][kParts][32];
};

// A lane's 16 elements of a block: runs of 16 bytes, a warp's side by side, where
// rows are 16-byte aligned (kVec); every 32nd element elsewhere.
template <typename T, bool kVec>
struct Lane {
  static constexpr int kWords = 16 * sizeof(T) / 4;
  uint32_t w[kWords];

  static __device__ __forceinline__ int index(int lane, int e) {
    constexpr int n = 16 / (int)sizeof(T);  // of a run
    return kVec ? (e / n) * (32 * n) + lane * n + e % n : e * 32 + lane;
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
      for (int q = 0; q < kWords / 4; ++q) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + at) + q * 32 + lane);
        w[q * 4] = v.x;
        w[q * 4 + 1] = v.y;
        w[q * 4 + 2] = v.z;
        w[q * 4 + 3] = v.w;
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
  __device__ __forceinline__ void take(const Ring<T>& ring, int stage, int lane) {
#pragma unroll
    for (int q = 0; q < Ring<T>::kParts; ++q) {
      const uint4 v = ring.part[stage][q][lane];
      w[q * 4] = v.x;
      w[q * 4 + 1] = v.y;
      w[q * 4 + 2] = v.z;
      w[q * 4 + 3] = v.w;
    }
  }
  __device__ __forceinline__ float2 pair(int p) const {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(w[2 * p]), __uint_as_float(w[2 * p + 1]));
    else
      return unpack2<T>(w[p]);
  }
  // The largest element, NaN if there is one; 16-bit types two at a time.
  __device__ __forceinline__ float most() const {
    if constexpr (sizeof(T) == 4) {
      auto v = [&](int i) { return __uint_as_float(w[i]); };
      float x = max3n(v(0), v(1), v(2)), y = max3n(v(3), v(4), v(5));
      x = max3n(max3n(x, v(6), v(7)), v(8), v(9));
      y = max3n(max3n(y, v(10), v(11)), v(12), v(13));
      return max3n(max3n(x, v(14), v(15)), y, y);
    } else {
      const uint32_t m = max2n(max2n(max2n(w[0], w[1]), max2n(w[2], w[3])),
                               max2n(max2n(w[4], w[5]), max2n(w[6], w[7])));
      const float2 v = unpack2<T>(m);
      return max3n(v.x, v.y, v.y);
    }
  }
  static __device__ __forceinline__ uint32_t max2n(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  // -inf as a number far below every maximum that Sums::add takes (kFar).
  __device__ __forceinline__ void lift() {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
      for (int p = 0; p < 8; ++p)
        asm("max.bf16x2 %0, %0, %1;" : "+r"(w[p]) : "r"(0xf149f149u));  // -1e30
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int p = 0; p < 8; ++p)
        asm("max.f16x2 %0, %0, %1;" : "+r"(w[p]) : "r"(0xfbfffbffu));  // -65504
    } else {
#pragma unroll
      for (int p = 0; p < 16; ++p) w[p] = __float_as_uint(fmaxf(__uint_as_float(w[p]), -1e30f));
    }
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

// A lane's running sums, all lanes of a warp with the same m. S is kept over
// ln(2): its terms are e^(x - m) t with the exponent t = (x - m) log2(e). The maximum is
// subtracted before the scaling. fma(x, log2(e), -m log2(e)) would save one of five
// packed instructions (4096 rows of bf16: 212 us in a burst, 216 so), but its exponents are
// all off by the rounding of m log2(e): by 1e-3 at |m| = 3e4, differently for each m that
// the running maximum took on, and by hundreds at |m| = 1e10.
template <typename T>
struct Running {
  // Below (or, bf16 and fp32, above) these, two values of T that differ do so by
  // 32 at least: the maximum's equals have the weight 1 and the others 1e-14 at most.
  static constexpr float kFarLow = std::is_same<T, __half>::value ? -60000.f : -0.9e30f;
  static constexpr float kFarHigh = 0.9e30f;
  float m = -INFINITY;
  float2 z = {0.f, 0.f}, s = {0.f, 0.f};

  // A block whose largest element over the warp is `most`.
  template <typename Block>
  __device__ __forceinline__ void add(Block& b, float most) {
    if (!(most <= m)) {
      if (most != most) most = INFINITY;
      const float d = fmaxf(m - most, kGone) * kLog2e, c = exp2_approx(d);
      s = make_float2((s.x + z.x * d) * c, (s.y + z.y * d) * c);
      z = make_float2(z.x * c, z.y * c);
      m = most;
    }
    if (m > kFarLow && m < kFarHigh) {
      b.lift();
      const float2 l2 = make_float2(kLog2e, kLog2e), nm = make_float2(-m, -m);
      // The block by itself first: a long row's sums then meet 8 times fewer
      // roundings, which for equal logits all go the same way (262656 sorted logits are
      // 1.1e-6 off without; 4096 rows of 151936 take 216 us without, 220 so).
      float2 zb, sb;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float2 t = mul2(add2(b.pair(p), nm), l2);
        const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
        zb = p == 0 ? e : add2(zb, e);
        sb = p == 0 ? mul2(e, t) : fma2(e, t, sb);
      }
      z = add2(z, zb);
      s = add2(s, sb);
    } else if (m > -INFINITY) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float2 v = b.pair(p);
        z.x += v.x == m ? 1.f : 0.f;
        z.y += v.y == m ? 1.f : 0.f;
      }
    }
  }
  // Over the warp.
  __device__ __forceinline__ Sums all() const {
    Sums r = {m, z.x + z.y, s.x + s.y};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      r.z += __shfl_xor_sync(0xffffffffu, r.z, o);
      r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    }
    r.s *= kLn2;
    return r;
  }
};

template <typename T>
struct Shared {
  Sums sums[kWarps];
  int sel[kMaxTopLogprobs];
  uint32_t thr;
  int n_sel, n_list, n_ties, last;
  union {
    Ring<T> ring[kWarps];                             // while the row is read
    struct {                                          // after it
      unsigned long long list[kList + kTies];
      uint32_t most[kThreads];
    };
  };
  union {  // [blocks], of the dynamic part
    float block_max[1];
    uint32_t keys[1];
  };
};

// The top_k elements of row x as (key, ~index) in sh.list, unsorted, from the
// block maxima in sh.keys; returns how many were listed (top_k at least).
template <typename T, bool kVec>
__device__ int list_top(Shared<T>& sh, const T* x, int V, int n_blocks, int top_k) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (warp == 0) {
    // top_k rounds: the largest key left, the first block of equals. The lanes
    // hold the keys of up to 512 blocks in registers, neighbours in a lane, so that
    // the first lane with the key has the first block.
    const int n = min(top_k, n_blocks);
    uint32_t k = 0;
    if (n_blocks <= 32 * 16) {
      const int per = (n_blocks + 31) / 32;
      uint32_t key[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        key[i] = i < per && lane * per + i < n_blocks ? sh.keys[lane * per + i] : 0;
      for (int r = 0; r < n; ++r) {
        uint32_t m[4] = {key[0], key[1], key[2], key[3]};
#pragma unroll
        for (int i = 4; i < 16; ++i) m[i % 4] = max(m[i % 4], key[i]);
        const uint32_t best = max(max(m[0], m[1]), max(m[2], m[3]));
        uint32_t at[4] = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) at[i % 4] |= key[i] == best ? 1u << i : 0u;
        const int first = __ffs((at[0] | at[1]) | (at[2] | at[3])) - 1;
        k = __reduce_max_sync(0xffffffffu, best);
        const int who = __ffs(__ballot_sync(0xffffffffu, best == k)) - 1;
        if (lane == who) sh.sel[r] = lane * per + first;
        const int gone = lane == who ? first : -1;
#pragma unroll
        for (int i = 0; i < 16; ++i) key[i] = i == gone ? 0u : key[i];
      }
    } else {
      for (int r = 0; r < n; ++r) {
        uint32_t best = 0;
        for (int i = lane; i < n_blocks; i += 32) best = max(best, sh.keys[i]);
        k = __reduce_max_sync(0xffffffffu, best);
        unsigned at = 0xffffffffu;
        if (best == k)
          for (int i = lane; i < n_blocks; i += 32)
            if (sh.keys[i] == k) at = min(at, (unsigned)i);
        const int b = (int)__reduce_min_sync(0xffffffffu, at);
        if (lane == 0) sh.sel[r] = b;
        if (b % 32 == lane) sh.keys[b] = 0;
        __syncwarp();
      }
    }
    if (lane == 0) {
      sh.n_sel = n;
      sh.thr = n == top_k ? k : 0;
      sh.n_list = sh.n_ties = 0;
    }
  }
  __syncthreads();
  const int n_sel = sh.n_sel;
  // f(v, at) for the lane's elements of every picked block, kBatch blocks of the
  // warp on their way at once
  auto each = [&](auto&& f) {
    constexpr int kBatch = 2;
    for (int b0 = warp; b0 < n_sel; b0 += kBatch * kWarps) {
      Lane<T, kVec> v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (b0 + j * kWarps < n_sel) v[j].load(x, sh.sel[b0 + j * kWarps] * kBlock, V, lane);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (b0 + j * kWarps < n_sel) f(v[j], sh.sel[b0 + j * kWarps] * kBlock);
    }
  };
  // the key of element e, 0 past the row's end
  auto key_of = [&](const Lane<T, kVec>& v, int at, int e) {
    const float2 p = v.pair(e / 2);
    return at + Lane<T, kVec>::index(lane, e) < V ? order_of(e % 2 ? p.y : p.x) : 0u;
  };
  auto collect = [&]() {
    const uint32_t thr = max(sh.thr, 1u);
    each([&](const Lane<T, kVec>& v, int at) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t k = key_of(v, at, e);
        if (k < thr) continue;
        const bool tie = k == thr;
        int* counter = tie ? &sh.n_ties : &sh.n_list;
        const int most = tie ? kTies : kList;
        // past its end the list does not count on: a mask of -inf can leave
        // thousands of ties
        if (*(volatile int*)counter > most) continue;
        const int i = atomicAdd(counter, 1);
        if (i < most)
          sh.list[tie ? kList + i : i] =
              ((unsigned long long)k << 32) | (uint32_t)~(at + Lane<T, kVec>::index(lane, e));
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
    each([&](const Lane<T, kVec>& v, int at) {
#pragma unroll
      for (int e = 0; e < 16; ++e) mine = max(mine, key_of(v, at, e));
    });
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
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 3 : 5)
    token_logprobs_kernel(TokenLogprobsArgs a, int splits, int n_blocks) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<T>& sh = *reinterpret_cast<Shared<T>*>(raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int r = blockIdx.x / splits, split = blockIdx.x % splits;
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)r * a.row;
  const int first = (int)((long long)n_blocks * split / splits);
  const int end = (int)((long long)n_blocks * (split + 1) / splits);
  float* keys = splits > 1 ? a.block_max + (size_t)r * n_blocks : sh.block_max;

  Running<T> run;
  // whole blocks of the warp through the ring, kStages - 1 ahead
  Ring<T>& ring = sh.ring[warp];
  const int whole = kVec ? min(end, a.V / kBlock) : 0;
  int b = first + warp;
  int ahead = b, stage = 0;
  const T* src = x + (size_t)b * kBlock + lane * (16 / (int)sizeof(T));
  auto fetch = [&](int st) {
    if (ahead < whole) {
      const uint32_t dst = smem_u32(&ring.part[st][0][lane]);
      if constexpr (sizeof(T) == 2)
        asm volatile(
            "cp.async.cg.shared.global [%0], [%1], 16;\n\t"
            "cp.async.cg.shared.global [%0 + 512], [%1 + 512], 16;" ::"r"(dst), "l"(src)
            : "memory");
      else
        asm volatile(
            "cp.async.cg.shared.global [%0], [%1], 16;\n\t"
            "cp.async.cg.shared.global [%0 + 512], [%1 + 512], 16;\n\t"
            "cp.async.cg.shared.global [%0 + 1024], [%1 + 1024], 16;\n\t"
            "cp.async.cg.shared.global [%0 + 1536], [%1 + 1536], 16;" ::"r"(dst), "l"(src)
            : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead += kWarps;
    src += kWarps * kBlock;
  };
  auto block = [&](Lane<T, kVec>& v) {
    const float most = warp_max_nan(v.most());
    if (a.top_k > 0 && lane == 0) keys[b] = most;
    run.add(v, most);
  };
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) fetch(st);
  for (; b < whole; b += kWarps) {
    fetch((stage + kStages - 1) % kStages);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    Lane<T, kVec> v;
    v.take(ring, stage, lane);
    stage = (stage + 1) % kStages;
    block(v);
  }
  for (; b < end; b += kWarps) {  // the row's last block, or rows off the 16-byte grid
    Lane<T, kVec> v;
    v.load(x, b * kBlock, a.V, lane);
    block(v);
  }
  const Sums mine = run.all();
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  Sums all = sh.sums[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) all = join(all, sh.sums[w]);
  if (splits > 1) {
    float* part = a.parts + ((size_t)r * splits + split) * 4;
    if (threadIdx.x == 0)
      *reinterpret_cast<float4*>(part) = make_float4(all.m, all.z, all.s, 0.f);
    __syncthreads();
    if (threadIdx.x == 0) {
      sh.last = count_arrival(&a.counters[r]) == splits - 1;
      if (sh.last) a.counters[r] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    const float4* parts = reinterpret_cast<const float4*>(a.parts) + (size_t)r * splits;
    float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    if (lane < splits) p = __ldcg(parts + lane);
    if (a.top_k > 0)
      for (int i = threadIdx.x; i < n_blocks; i += kThreads) sh.block_max[i] = __ldcg(keys + i);
    all = {p.x, p.y, p.z};
    for (int i = lane + 32; i < splits; i += 32) {
      p = __ldcg(parts + i);
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
  for (int i = threadIdx.x; i < n_blocks; i += kThreads) sh.keys[i] = order_of(sh.block_max[i]);
  __syncthreads();
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
  const size_t bytes = sizeof(Shared<T>) + (size_t)(a.top_k > 0 ? n_blocks : 0) * 4;
  const bool vec = ((uintptr_t)a.logits & 15) == 0 &&
                   (a.R == 1 || a.row * (long long)sizeof(T) % 16 == 0);
  const auto kern = vec ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern),
                                       (int)(sizeof(Shared<T>) + kMaxBlocks * 4));
  if (e == cudaSuccess)
    e = launch_k(kern, dim3((unsigned)(a.R * splits)), dim3(kThreads), bytes, s, a, splits,
                 n_blocks);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

int blocks_of(int V) { return (V + kBlock - 1) / kBlock; }

}  // namespace

// CTAs of a row: two on each SM in all at most, a block for each warp at least
// (33 rows of fp32, top 20, a ring of four: 17.0 us with 8 CTAs a row, 18.2 with 17; 256 of bf16: 29 with
// one, 35 with two to four). Between two and four rows an SM, where one CTA a row
// leaves the last ones alone, two: 400 rows 45 us, 52 with one.
int token_logprobs_splits(int R, int V, int num_sms) {
  const int most = (blocks_of(V) + kWarps - 1) / kWarps;
  int want = 2 * num_sms / max(R, 1);
  if (want < 1) want = R < 4 * num_sms ? 2 : 1;
  return want < most ? want : most;
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
  a.block_max = a.parts + (size_t)a.R * splits * 4;
  if (a.elem == kElemBf16) return launch_one<__nv_bfloat16>(a, splits, n_blocks, s);
  if (a.elem == kElemF16) return launch_one<__half>(a, splits, n_blocks, s);
  return launch_one<float>(a, splits, n_blocks, s);
}

}  // namespace afd
