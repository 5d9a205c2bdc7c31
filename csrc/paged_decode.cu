// Attention of one new token per sequence over the paged KV cache, split over
// the cache's length and joined in the same launch.
//
//   out[b, h] = sum_j p_j v_j, p = softmax over j < seq_lens[b] of
//   q[b, h] . k_j * scale, with h's kv head h / G, G = nq / nkv
//
// What bounds it is reading K and V once: 4 G flops an element of K or V, a
// hundredth of what the tensor cores have over the HBM's rate. So the layout serves
// the loads, and the products use the warp-level MMA, whose operands and
// results stay in the registers of one warp: no barrier between warps, no
// round trip through TMEM, and a running maximum of each warp's own.
//
// A warp takes blocks of 16 keys (a page holds a whole number of them) through
// a ring of its own in shared memory, which its lane 0 refills by TMA as soon as
// the block is consumed. For a block, with the keys as the rows of the MMA:
//
//   S^T [16 keys x 8 heads]  = K [16 x D] Q^T          (K by ldmatrix)
//   O^T [D x 8 heads]       += V^T [D x 16] P^T        (V by ldmatrix.trans)
//
// S^T's result layout turns into P^T's operand layout by one 8x8 transpose
// (movmatrix), and the heads of S^T, P^T and O^T lie in the same lanes, so
// maxima and rescales need no exchange. G up to 16 heads take one or two
// tiles of 8; more take several passes over K and V.
//
// P enters the second product as the sum of two values of the input type (high
// part and remainder), so that the weights keep 16 bits and more: the
// tensor pipe has the room, and the output is then rounded once, as the formula is.
//
// Split: the 16-key blocks of all (sequence, kv head) items, in order, are cut
// into equal ranges, one per CTA, and a range end near an item's end moves there. Over
// long caches the ranges stay equal (16 sequences of 20000..40960: 399 blocks at most,
// 392 on average; 150.5 us for 950 MB, 6.3 TB/s). Over short ones moving saves cuts but
// leaves ranges uneven (32 sequences of 128..4096: 60 blocks at most, 33 on average, 110 and
// 66 on an SM; 22.5 us, where the bytes take 12.3). A CTA joins its 4 warps in shared memory; an item cut by a range
// end leaves fp32 partials (O, maximum, sum) in the workspace, and the CTA
// that counts the last of its parts joins them, in the order of the parts.

#include <string.h>

#include <atomic>

#include "ragged.cuh"

namespace afd {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kBlk = 16;                 // keys of a block
// Ring depth of a warp: 128 KB on their way to an SM. With three (192 KB) the
// SMs' shares of the HBM's rate drift apart: 154 us against 150 for 950 MB.
constexpr int kStages = 2;
constexpr int kCtasPerSm = 2;            // one joins and looks up while the other loads

// Units of work: blocks, and kItemCost more for an item (its queries, the join
// of the warps). A range holds an equal share of them, at least kMinRange (short
// sequences stay whole). A range end near an item's end is moved there, within
// half a range where ranges are short (up to kShortRange) and within kSnap units
// where they are long: a cut costs a join through the workspace, an uneven range
// what it has more.
constexpr int kItemCost = 4;
constexpr int kMinRange = 20;
constexpr int kShortRange = 40;
constexpr int kSnap = 8;

template <int D>
struct Dec {
  static constexpr int kBox = kBlk * 128;             // one 128-byte wide box
  static constexpr int kTile = kBlk * D * 2;          // K or V of a block
  static constexpr int kStage = 2 * kTile;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kTasks = (2 * D + kThreads - 1) / kThreads;  // float4 of 8 heads a thread joins
  static constexpr int kJoin = kWarps * 8 * D * 4;
  static constexpr int kBytes = kRing + kJoin + kWarps * (8 * kStages + 64 + 4) + 128;
};

// A part in the workspace: (maximum, sum) of its heads, then their O.
template <int D, int NT>
struct Part {
  static constexpr int kHeads = 8 * NT;
  static constexpr int kStats = kHeads * 8;
  static constexpr int kBytes = kStats + kHeads * D * 4;
};

// Float index of (warp, head, dim) in the join buffer: the heads of a quarter
// warp start 8 banks apart.
template <int D>
__device__ __forceinline__ int join_at(int w, int h, int d) {
  return (w * 8 + h) * D + (d ^ ((h >> 1) * 8));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Bulk copy of `bytes` (a multiple of 16, both ends 16-byte aligned).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Four output values of a head, from their weighted sum and the weights' sum.
template <typename T, int D>
__device__ __forceinline__ void store_out(const PagedDecodeArgs& a, int b, int h, int d, float4 acc,
                                          float l) {
  const float inv = 1.f / l;
  uint2 v = make_uint2(0u, 0u);  // every weight 0
  if (!(l == 0.f))
    v = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + ((size_t)b * a.nq + h) * D + d) = v;
}

// A place in the order of all work: item (sequence b, kv head and head group
// `sub`), the item's extent [begin, end) in units of blocks, kItemCost of them
// for the item itself, and the portion [j0, j1) of its blocks that is this CTA's.
// `before` counts the CTA's blocks of earlier items: block j goes to warp
// (before + j - j0) % kWarps.
struct Cursor {
  int b, sub, len, len_next;
  int begin, end;
  int j0, j1, before;
};

struct Place {  // of a range end: the item that it falls into, moved to an end of it if near
  int b, sub, len;
  int begin, end, at;
};

}  // namespace

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tk,
                        const __grid_constant__ CUtensorMap tv, PagedDecodeArgs a, int groups) {
  using C = Dec<D>;
  extern __shared__ __align__(1024) uint8_t smem[];  // whole swizzle atoms
  float* join = reinterpret_cast<float*>(smem + C::kRing);           // [warps][8][D], join_at
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kRing + C::kJoin);  // [warps][stages]
  float2* ml = reinterpret_cast<float2*>(full + kWarps * kStages);   // [warps][8]
  int* scan = reinterpret_cast<int*>(ml + kWarps * 8);               // [warps]
  Place* place = reinterpret_cast<Place*>(scan + kWarps);            // [2]: of r0, r1
  uint64_t* part_bar = reinterpret_cast<uint64_t*>(place + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(part_bar + 1);
  volatile int* joins_item = abort_flag + 1;                         // [2]
  volatile int* any_empty = joins_item + 2;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = a.nq / a.nkv, subs = a.nkv * groups;
  const int most = a.max_pages * a.page_size;
  if (threadIdx.x < kWarps * kStages) mbar_init(&full[threadIdx.x], 1);
  if (threadIdx.x == 0) {
    mbar_init(part_bar, 1);
    *abort_flag = 0;
    *any_empty = 0;
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  fence_barrier_init();
  pdl_wait();
  pdl_trigger();

  // ---- the extent of the work: a scan over the sequences
  auto extent = [](int len) { return len > 0 ? (len + kBlk - 1) / kBlk + kItemCost : 0; };
  const int chunk = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(a.B, (int)threadIdx.x * chunk), b1 = min(a.B, b0 + chunk);
  int mine = 0;
  bool empty = false;
  for (int b = b0; b < b1; ++b) {
    const int len = checked_len(a.seq_lens[b], most, a.status, 221);
    mine += extent(len) * subs;
    empty |= len == 0 && b % gridDim.x == blockIdx.x;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  if (empty) *any_empty = 1;  // read after the next barrier
  int total = 0, before = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = total;
    total += scan[w];
  }
  before += upto - mine;
  const int range = max(kMinRange, (int)((total + gridDim.x - 1) / gridDim.x));
  // a range end this near to an item's is moved there
  const int snap = range <= kShortRange ? range / 2 : kSnap;
  // An item is cut at the multiples of `range` inside it that are not near its
  // ends: CTA `first_cta` has its first part, the p-th after it part p.
  auto first_cta = [&](int begin) { return (begin + snap) / range; };
  auto parts_of = [&](int begin, int end) {
    return (end - snap - 1) / range - first_cta(begin) + 1;
  };
  using P = Part<D, NT>;
  auto part_at = [&](int slot) { return reinterpret_cast<uint8_t*>(a.parts) + (size_t)slot * P::kBytes; };
  int part_phase = 0;
  const int id = blockIdx.x;

  uint8_t* ring = smem + warp * kStages * C::kStage;
  uint64_t* bar = full + warp * kStages;
  const float scale_log2 = a.scale * 1.4426950408889634f;
  int issued = 0, used = 0;
  bool ok = true;
  const int raw0 = (int)min((long long)id * range, (long long)total);
  const int raw1 = total - raw0 > range ? raw0 + range : total;
  for (int e = 0; e < 2; ++e) {
    const int r = e == 0 ? raw0 : raw1;
    if (r < before || r - before >= mine) continue;
    int at = before;
    for (int b = b0; b < b1; ++b) {
      const int len = checked_len(a.seq_lens[b], most, nullptr, 0);
      const int ext = extent(len);
      if (r - at < ext * subs) {
        Place p;
        p.b = b;
        p.len = len;
        p.sub = (r - at) / ext;
        p.begin = at + p.sub * ext;
        p.end = p.begin + ext;
        p.at = r - p.begin <= snap ? p.begin : p.end - r <= snap ? p.end : r;
        place[e] = p;
        break;
      }
      at += ext * subs;
    }
  }
  if (threadIdx.x == 0 && raw1 == total) place[1].at = total;
  __syncthreads();
  const int r0 = raw0 < total ? place[0].at : total, r1 = place[1].at;

  // the item after `c` and this CTA's portion of it
  auto take = [&](Cursor& c) {
    c.j0 = r0 > c.begin ? r0 - c.begin - kItemCost : 0;
    c.j1 = min(c.end, r1) - c.begin - kItemCost;
  };
  auto next_item = [&](Cursor& c) {
    c.before += c.j1 - c.j0;
    c.begin = c.end;
    if (++c.sub == subs) {
      c.sub = 0;
      do {
        ++c.b;
        c.len = c.b < a.B ? checked_len(c.len_next, most, nullptr, 0) : 1;
        c.len_next = c.b + 1 < a.B ? a.seq_lens[c.b + 1] : 0;
      } while (c.len == 0);
    }
    c.end = c.begin + extent(c.len);
    take(c);
  };
  Cursor ic;
  if (r0 < r1) {
    const Place p = place[0];
    ic.b = p.b;
    ic.sub = p.sub;
    ic.len = p.len;
    ic.len_next = p.b + 1 < a.B ? a.seq_lens[p.b + 1] : 0;
    ic.begin = p.begin;
    ic.end = p.end;
    ic.before = 0;
    if (r0 == p.end) {
      ic.j0 = ic.j1 = 0;
      next_item(ic);
    } else {
      take(ic);
    }
  }
  Cursor cc = ic;

  // ---- the warp's loads, kStages blocks ahead
  auto first_block = [&](const Cursor& c) { return c.j0 + ((warp - c.before) & (kWarps - 1)); };
  int ij = 0, held = 0, page = 0, row = 0;
  bool more = r0 < r1;
  // each lane holds the page of one of the next 32 blocks
  auto look_up = [&]() {
    const int key = (ij + lane * kWarps) * kBlk;
    held = 0;
    if (more && key < ic.j1 * kBlk) {
      page = a.page_table[(size_t)ic.b * a.table_row + key / a.page_size];
      row = (ic.sub / groups) * a.page_size + key % a.page_size;
    }
  };
  auto find = [&]() {  // the item of the next block to load
    while (more && ij >= ic.j1) {
      if (ic.end >= r1) {
        more = false;
      } else {
        next_item(ic);
        ij = first_block(ic);
      }
    }
    look_up();
  };
  auto issue = [&]() {
    if (!more) return;
    const int st = issued % kStages;
    const int pg = __shfl_sync(0xffffffffu, page, held), rw = __shfl_sync(0xffffffffu, row, held);
    if (lane == 0) {
      if (pg < 0 || pg >= a.num_pages)  // the copies fill with zeros
        report_status(a.status, kBoundsViolation, 222);
      uint8_t* dst = ring + st * C::kStage;
      mbar_arrive_expect_tx(&bar[st], C::kStage);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        tma_load_3d(dst + c * C::kBox, &tk, &bar[st], c * 64, rw, pg);
        tma_load_3d(dst + C::kTile + c * C::kBox, &tv, &bar[st], c * 64, rw, pg);
      }
    }
    ++issued;
    ij += kWarps;
    if (ij >= ic.j1)
      find();
    else if (++held == 32)
      look_up();
  };
  if (more) ij = first_block(ic);
  find();
  for (int s = 0; s < kStages; ++s) issue();

  // Q^T as the B operand: head lane / 4, dims 2 (lane % 4) + {0, 1, 8, 9} of 16
  uint32_t qf[NT][D / 16][2];
  auto load_q = [&](const Cursor& c) {
    const int grp = c.sub % groups, h0 = (c.sub / groups) * G + grp * 8 * NT;
    const int heads = min(8 * NT, G - grp * 8 * NT);
    const T* q = reinterpret_cast<const T*>(a.q) + (size_t)c.b * a.q_row + (size_t)h0 * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qf[n][kk][e] = n * 8 + lane / 4 < heads
                             ? *reinterpret_cast<const uint32_t*>(
                                   q + (n * 8 + lane / 4) * D + kk * 16 + (lane % 4) * 2 + e * 8)
                             : 0u;
  };
  if (r0 < r1) load_q(cc);

  // ---- the items of the range
  const Cursor head = cc;
  while (r0 < r1) {
    const int grp = cc.sub % groups, h0 = (cc.sub / groups) * G + grp * 8 * NT;
    const int heads = min(8 * NT, G - grp * 8 * NT);
    // lane: heads 2 (lane % 4) + {0, 1} of each tile
    float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][d][e] = 0.f;
    }
    for (int j = first_block(cc); j < cc.j1; j += kWarps) {
      const int st = used % kStages;
      if (ok && !__all_sync(0xffffffffu, mbar_wait(&bar[st], (used / kStages) & 1, abort_flag,
                                                   a.status, 223)))
        ok = false;
      const uint32_t ks = smem_u32(ring + st * C::kStage), vs = ks + C::kTile;
      const int key0 = j * kBlk;
      // two chains of products, the even and the odd 16 dims
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
      {
        const int r = (lane / 8 % 2) * 8 + lane % 8;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          const int ch = (kk % 4) * 2 + lane / 16;
          ldsm4(ks + (kk / 4) * C::kBox + r * 128 + ((ch ^ (r & 7)) << 4), kf);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma16816<T>(kk % 2 ? s2[n] : s[n], kf, qf[n][kk][0], qf[n][kk][1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
      if (key0 + kBlk > cc.len) {
        // keys past the end: no weight, and finite values for it to meet
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + lane / 4 + (e / 2) * 8 >= cc.len) s[n][e] = -INFINITY;
        for (int i = lane; i < kBlk * D / 8; i += 32) {
          const int r = i / 8 % kBlk;
          if (key0 + r >= cc.len)
            *reinterpret_cast<uint4*>(ring + st * C::kStage + C::kTile + i * 16) =
                make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[4];
        // rounded here, not within a multiply-add, so that the largest one's x - m is 0
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __fmul_rn(s[n][e], scale_log2);
        // the maximum moves only when it grows by more than 8 (powers of two)
        const bool grow = fmaxf(x[0], x[2]) > m[n][0] + 8.f || fmaxf(x[1], x[3]) > m[n][1] + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(m[n][e], fmaxf(x[e], x[e + 2]));
#pragma unroll
            for (int f = 4; f < 32; f <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, f));
            const float c = mx == -INFINITY ? 1.f : exp2_approx(m[n][e] - mx);
            m[n][e] = mx;
            l[n][e] *= c;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[n][d][e] *= c;
              o[n][d][e + 2] *= c;
            }
          }
        }
        float p[4], r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // a masked key weighs nothing; a score that is NaN, which no maximum holds, stays
          p[e] = x[e] == -INFINITY ? 0.f : exp2_approx(x[e] - m[n][e & 1]);
          r[e] = p[e] - to_f(from_f<T>(p[e]));
        }
        l[n][0] += p[0] + p[2];
        l[n][1] += p[1] + p[3];
        ph[n][0] = transpose8(pack2<T>(p[0], p[1]));
        ph[n][1] = transpose8(pack2<T>(p[2], p[3]));
        pl[n][0] = transpose8(pack2<T>(r[0], r[1]));
        pl[n][1] = transpose8(pack2<T>(r[2], r[3]));
      }
      {
        const int r = (lane / 16) * 8 + lane % 8;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t vf[4];
          const int ch = (d % 4) * 2 + (lane / 8) % 2;
          ldsm4_t(vs + (d / 4) * C::kBox + r * 128 + ((ch ^ (r & 7)) << 4), vf);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816<T>(o[n][d], vf, ph[n][0], ph[n][1]);
            mma16816<T>(o[n][d], vf, pl[n][0], pl[n][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the block
      ++used;
      issue();
    }

    // ---- join the warps; the next item's queries are on their way meanwhile
    const Cursor item = cc;
    const bool more_items = cc.end < r1;
    if (more_items) {
      next_item(cc);
      load_q(cc);
    }
    const bool cut = item.begin < r0 || item.end > r1;
    uint8_t* part = part_at(item.begin < r0 ? 2 * id : 2 * id + 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      __syncthreads();  // the buffer's last readers are done
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = (lane % 4) * 2 + e;
#pragma unroll
        for (int f = 4; f < 32; f <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], f);
        if (lane < 4) ml[warp * 8 + h] = make_float2(m[n][e], l[n][e]);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          join[join_at<D>(warp, h, d * 16 + lane / 4)] = o[n][d][e];
          join[join_at<D>(warp, h, d * 16 + 8 + lane / 4)] = o[n][d][e + 2];
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * D / 4; i += kThreads) {
        const int h = i / (D / 4), d = i % (D / 4) * 4, hd = n * 8 + h;
        if (hd >= heads) break;
        float M = -INFINITY, lsum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w * 8 + h].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 s = ml[w * 8 + h];
          // by the sum: of a warp whose scores are all NaN the maximum is -inf too
          const float c = s.y == 0.f ? 0.f : exp2_approx(s.x - M);
          const float4 v = *reinterpret_cast<const float4*>(join + join_at<D>(w, h, d));
          lsum += s.y * c;
          acc.x += v.x * c;
          acc.y += v.y * c;
          acc.z += v.z * c;
          acc.w += v.w * c;
        }
        if (cut) {
          *reinterpret_cast<float4*>(part + P::kStats + (hd * D + d) * 4) = acc;
          if (d == 0) reinterpret_cast<float2*>(part)[hd] = make_float2(M, lsum);
        } else {
          store_out<T, D>(a, item.b, h0 + hd, d, acc, lsum);
        }
      }
    }
    if (!more_items) break;
  }

  // ---- cut items: whoever counts the last part joins them all. The
  // first and the last item of a range can be cut.
  const Cursor& tail = cc;
  const bool cut0 = r0 < r1 && (head.begin < r0 || head.end > r1);
  const bool cut1 = r0 < r1 && tail.begin > head.begin && tail.end > r1;
  if (cut0 || cut1) {
    fence_proxy_async_global();  // bulk copies read the parts
    __syncthreads();
    if (threadIdx.x < 2) {
      const Cursor& c = threadIdx.x == 0 ? head : tail;
      int last = 0;
      if (threadIdx.x == 0 ? cut0 : cut1) {
        int* counter = a.counters + first_cta(c.begin);
        last = count_arrival(counter) == parts_of(c.begin, c.end) - 1;
        if (last) *counter = 0;
      }
      joins_item[threadIdx.x] = last;
    }
    __syncthreads();
    for (int e = 0; e < 2; ++e) {
      if (!joins_item[e]) continue;
      const Cursor& c = e == 0 ? head : tail;
      const int c0 = first_cta(c.begin), parts = parts_of(c.begin, c.end);
      const int grp = c.sub % groups, h0 = (c.sub / groups) * G + grp * 8 * NT;
      const int heads = min(8 * NT, G - grp * 8 * NT);
      // the parts into the ring (every load of it has been consumed), as many
      // at once as it holds
      constexpr int kBatch = C::kRing / P::kBytes;
      const uint32_t bytes = P::kStats + heads * D * 4;
      float M[NT * C::kTasks], lsum[NT * C::kTasks];
      float4 acc[NT * C::kTasks];
#pragma unroll
      for (int t = 0; t < NT * C::kTasks; ++t) {
        M[t] = -INFINITY;
        lsum[t] = 0.f;
        acc[t] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      for (int p0 = 0; p0 < parts; p0 += kBatch) {
        const int n = min(kBatch, parts - p0);
        __syncthreads();
        if (threadIdx.x == 0) {
          fence_proxy_async_global();
          mbar_arrive_expect_tx(part_bar, n * bytes);
          for (int p = 0; p < n; ++p) {
            const int k = p0 + p;
            bulk_load(smem + p * P::kBytes, part_at(k == 0 ? 2 * c0 + 1 : 2 * (c0 + k)), bytes,
                      part_bar);
          }
        }
        if (!mbar_wait(part_bar, part_phase, abort_flag, a.status, 225)) ok = false;
        part_phase ^= 1;
#pragma unroll
        for (int t = 0; t < NT * C::kTasks; ++t) {
          const int i = t * kThreads + threadIdx.x, hd = i / (D / 4), d = i % (D / 4) * 4;
          if (hd >= heads) break;
          float m_new = M[t];
          for (int p = 0; p < n; ++p)
            m_new = fmaxf(m_new, reinterpret_cast<const float2*>(smem + p * P::kBytes)[hd].x);
          const float f0 = M[t] == -INFINITY ? 0.f : exp2_approx(M[t] - m_new);
          M[t] = m_new;
          lsum[t] *= f0;
          acc[t] = make_float4(acc[t].x * f0, acc[t].y * f0, acc[t].z * f0, acc[t].w * f0);
          for (int p = 0; p < n; ++p) {
            const uint8_t* at = smem + p * P::kBytes;
            const float2 s = reinterpret_cast<const float2*>(at)[hd];
            const float4 v = *reinterpret_cast<const float4*>(at + P::kStats + (hd * D + d) * 4);
            const float f = s.y == 0.f ? 0.f : exp2_approx(s.x - m_new);
            lsum[t] += s.y * f;
            acc[t].x += v.x * f;
            acc[t].y += v.y * f;
            acc[t].z += v.z * f;
            acc[t].w += v.w * f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT * C::kTasks; ++t) {
        const int i = t * kThreads + threadIdx.x, hd = i / (D / 4), d = i % (D / 4) * 4;
        if (hd < heads) store_out<T, D>(a, c.b, h0 + hd, d, acc[t], lsum[t]);
      }
    }
  }

  // sequences without a key: zeros
  if (*any_empty)
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      if (checked_len(a.seq_lens[b], most, nullptr, 0) == 0)
        for (int i = threadIdx.x; i < a.nq * D / 8; i += kThreads)
          reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + (size_t)b * a.nq * D)[i] =
              make_uint4(0, 0, 0, 0);
  if (!ok && lane == 0) {
    // loads that a failed wait left in flight must land before the CTA exits
    volatile int no_abort = 0;
    for (int j = max(0, issued - kStages); j < issued; ++j)
      mbar_wait(&bar[j % kStages], (j / kStages) & 1, &no_abort, nullptr, 224, 100000000ull);
    mbar_wait(part_bar, part_phase ^ 1, &no_abort, nullptr, 226, 100000000ull);
  }
}

// ============================================================ host side ===

template <typename T, int D, int NT>
static int launch_one(const PagedDecodeArgs& a, int grid, int groups, const CUtensorMap& tk,
                      const CUtensorMap& tv, cudaStream_t s) {
  const auto kern = paged_decode_kernel<T, D, NT>;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), Dec<D>::kBytes);
  int dev = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return 4000 + (int)e;
  // room for both CTAs of an SM, asked for once per device
  static std::atomic<uint64_t> asked{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (!(asked.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e == cudaSuccess)
    e = launch_k(kern, dim3(grid), dim3(kThreads), Dec<D>::kBytes, s, tk, tv, a, groups);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

long long paged_decode_part_bytes(int nq, int nkv, int D, int num_sms) {
  return 2ll * num_sms * kCtasPerSm * (nq / nkv > 8 ? 16 : 8) * (8 + 4 * D);
}

int paged_decode_counters(int num_sms) { return num_sms * kCtasPerSm; }

int launch_paged_decode(const PagedDecodeArgs& a, int num_sms, cudaStream_t s) {
  if (a.B == 0) return 0;
  const int grid = num_sms * kCtasPerSm;
  CUtensorMap tk, tv;
  // pool [pages, nkv * page_size, D]: a box is the 16 rows of a block
  const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.nkv * a.page_size, (uint64_t)a.num_pages};
  const uint64_t str[2] = {(uint64_t)a.D * 2, (uint64_t)a.page_stride * 2};
  const uint32_t box[3] = {64, kBlk, 1};
  if (int e = encode_map16(&tk, a.k_pages, a.elem, 3, dims, str, box)) return e;
  if (int e = encode_map16(&tv, a.v_pages, a.elem, 3, dims, str, box)) return e;
  const int G = a.nq / a.nkv, groups = (G + 15) / 16;
#define AFD_DECODE(T, D)                                            \
  (G > 8 ? launch_one<T, D, 2>(a, grid, groups, tk, tv, s)          \
         : launch_one<T, D, 1>(a, grid, groups, tk, tv, s))
  if (a.elem == kElemBf16)
    return a.D == 128 ? AFD_DECODE(__nv_bfloat16, 128) : AFD_DECODE(__nv_bfloat16, 64);
  return a.D == 128 ? AFD_DECODE(__half, 128) : AFD_DECODE(__half, 64);
#undef AFD_DECODE
}

}  // namespace afd
