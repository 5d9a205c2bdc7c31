// Causal GQA attention of packed queries over packed keys or over the paged
// cache, on the 5th-generation tensor cores.
//
//   out[r, h] = sum_j p_j v_j,  p = softmax over the visible keys j <= pos(r)
//               of q[r, h] . k_j * scale, with h's kv head h / G, G = nq / nkv
//
// The G heads that share a kv head share every K and V row, so a row tile of
// the first product holds 128 / G tokens x G heads of one sequence: a short
// prompt still fills the tile, and only the keys that its few tokens see are
// visited (a 128-token tile of one head would spend half of its last key tile
// on the mask). One block is two such row tiles, A and B, of consecutive
// tokens, which share every K and V tile in shared memory.
//
// Steps of 64 keys. For row tile X, S_X = Q_X K^T (M 128, N 64) and
// O_X += P_X V (P from TMEM) accumulate in TMEM; S and P of consecutive steps
// take two buffers in turn, so the product S_X(i+1) runs beside the softmax of
// step i. With one buffer (S freed once the softmax holds it, P apart) the four
// long prompts below took 927 us.
//
//   warp 0      work items, TMA producer: Q tiles, then K and V rings of 4 steps
//   warp 1      TMEM owner (512 columns) and MMA issuer
//   warps 2..5  softmax of row tile A, warps 6..9 of row tile B (a row a thread)
//
// Issue order of the MMA warp, i the step:  P_A(i) V | S_B(i+1) | P_B(i) V |
// S_A(i+2).  S_X(i+2) overwrites P_X(i): it waits for the commit of P_X(i) V,
// half a step old by then.
//
// The running maximum is raised only when a row's maximum grows by more than 8
// (in powers of two): P then holds values up to 256, exact in the ratio O / l,
// and O is rescaled in TMEM only in such steps. The exponents are fma(s, c, -m) with
// c = scale log2(e) and m = c max(s) rounded: every weight of a row has the same factor
// for that rounding. Where it could leave the range (|m| from 2^26 on, scores that only
// an overflow makes) it is taken out again, see Ref; without that the 32 prompts below
// take 71.3 us, 72.6 so, and the 4 long ones 876, 882. P is rounded to the input type
// for the second product; maxima, sums and both accumulators are fp32. With P as high
// part and remainder, as in paged_decode.cu, the second product runs twice in the chain
// that bounds a step: 32 prompts 92 us, 4 long ones 1220 (73 and 884 with P rounded).
// The error against 64 bits is then the output's own rounding, 0.0016 in bf16 and 0.00021
// in fp16; with P rounded it is 0.0019..0.0022 and 0.00029.
//
// TMEM columns: S_A [0,128), S_B [128,256) (two buffers of 64; P over the first
// 32 of each), O_A [256,256+D), O_B [384,384+D).
//
// Persistent CTAs take items (block of a sequence, kv head) in turn from a
// counter that wraps to zero with the last fetch of a launch. Slot s of the
// blocks belongs to the last sequence i with cu[i] / TB + i <= s: that leaves
// at least ceil(length / TB) slots for each sequence without a prefix sum over
// lengths, and a sequence's longest-running blocks come first.
//
// Where the blocks are too few for the SMs (a chunk of few tokens over a long
// cache), the keys of a block are cut into equal parts, as many as fill the SMs
// once, of 8 steps at least; each part leaves O, maximum and sum in fp32 and a
// second kernel joins the rows. 4 chunks of 16 tokens over 20000 positions: 45 us
// split, 260 whole; parts of 6 steps at least do no better, of 12 worse (4 x 16
// over 2000: 24 us, 18.5 with 8).
//
// Measured (bf16, 32 heads over 4 of 128): 4 prompts of 2338..8192 tokens, 991
// GFLOP visible, 884 us, 1.12 PF/s; 32 prompts of 5..1021, 73 us (short bursts; 913 and
// 81 in calls repeated for half a second, at lower clocks). A step of both row
// tiles takes 1820 cycles, for 1024 of products and as many of exponentials (4096
// tokens: tensor pipe 57%, special function units 61%, issue slots 40%, reads of
// shared memory by the MMAs 57%): none is full, what is left is the chain of a
// tile's softmax, P V, and S two steps on, between the two tiles. Other orders of the
// MMAs (S_X(i+2) right behind P_X(i) V; S before P V) take 970..1030 us. One row tile a
// CTA, two CTAs an SM, takes 940 us, and 68 for the 32 prompts, whose 5 steps a block
// hide less of each block's start and end.

#include <string.h>

#include <algorithm>

#include "ragged.cuh"

namespace afd {

namespace {

constexpr int kRows = 128;    // rows of a tile (TMEM lanes)
constexpr int kKeys = 64;     // keys of a step
constexpr int kStages = 4;    // K and V ring depth
constexpr int kThreads = 320;

// Parts of an item's keys: at most kMaxParts, of kMinPart steps at least.
constexpr int kMaxParts = 32;
constexpr int kMinPart = 8;

// What a row's weights are relative to: 2^(m + r), m = c s rounded for its largest score s
// and r the rounding where |m| is large (up to 2 left in below that), else 0.
struct Ref {
  float m, r;
};
constexpr float kFar = 67108864.f;  // 2^26

__device__ __forceinline__ Ref ref_of(float s, float c) {
  const float m = s * c;
  return {m, fabsf(m) >= kFar && fabsf(m) < INFINITY ? fmaf(s, c, -m) : 0.f};
}
// Exponent of a / b, -inf where a has seen no key.
__device__ __forceinline__ float over(const Ref& a, const Ref& b) { return (a.m - b.m) + (a.r - b.r); }

struct Item {
  int steps;    // 64-key steps of this part; 0: no key; -1: no more work
  int parts;    // number of parts | this one << 8
  int row0;     // query row of the block's first token
  int tokens;   // tokens of the sequence from there on (may exceed the block)
  int pos0;     // position of the first token, from the part's first key on
  int kvh;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 32 lanes x 32 bit, 64 consecutive columns per thread: two loads, one wait.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]),
        "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]),
        "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]),
        "=r"(r[62]), "=r"(r[63])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_st16_raw(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32"
      " [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
        "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Halves of the shared-memory matrix descriptors (umma_desc_sw128 and
// umma_desc_sw128_mn): the low one moves with the address, so that the issuing
// thread, whose own latency every step passes through, adds one constant per operand.
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr, uint32_t lbo) {
  return ((smem_addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);  // SBO, version, 128 B swizzle

// D (TMEM) (+)= A x B, both in shared memory.
template <bool kAccumulate>
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                        uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %4};\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "n"(kAccumulate ? 1 : 0)
      : "memory");
}

// D (TMEM) (+)= A (TMEM, 128 lanes x 16 elements) x B (shared memory).
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(accumulate)
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t idesc16(int M, int N, bool b_mn_major) {
  uint32_t d = umma_idesc_bf16(M, N, b_mn_major);
  // formats of A (bits 7..9) and B (10..12): 1 = bf16, 0 = fp16
  if (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value) d &= ~((1u << 7) | (1u << 10));
  return d;
}

template <int D>
struct Smem {
  static constexpr int kBoxes = D / 64;                 // 128-byte wide boxes of a row
  static constexpr int kQTile = kRows * D * 2;          // one row tile
  static constexpr int kQBox = kRows * 128;
  static constexpr int kKvTile = kKeys * D * 2;         // K or V of one step
  static constexpr int kKvBox = kKeys * 128;
  static constexpr int kStage = 32 * 128;               // a warp's output rows, 64 dims
  static constexpr int kBytes =
      2 * kQTile + 2 * kStages * kKvTile + 8 * kStage + 1024 /*align*/ + 512;
};

// What the softmax warps (256 threads) do while the first item's queries and keys
// are on their way: check the query offsets, and store zeros, each CTA its share, to the
// rows that no item stores: those before the first offset, or all rows where offsets
// decrease. Such a list gives some rows two owners and others none, so then (true)
// no item stores anything. Every CTA reads the whole list and comes to the same
// answer: n / 256 loads a thread, against n * nkv / 148 items of a microsecond or more.
// A call, so that the loop behind it keeps its registers (inlined, it spilled 48 bytes).
__device__ __noinline__ bool settle_offsets(const int* cu_q, int n, int T, int nq, int D, void* out,
                                            int* n_parts, int* status) {
  const int id = threadIdx.x - 64;
  bool outside = false, down = false;
  for (int i = id; i <= n; i += 256) {
    const int c = cu_q[i], next = cu_q[min(i + 1, n)];
    outside |= c < 0 || c > T;
    down |= min(max(next, 0), T) < min(max(c, 0), T);
  }
  if ((outside || down) && blockIdx.x == 0) report_status(status, kBoundsViolation, 210);
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, 1, 256, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)down)
      : "memory");
  const size_t rows = (size_t)(any ? T : min(max(cu_q[0], 0), T)) * nq;
  const size_t first = (size_t)blockIdx.x * 256 + id, step = (size_t)gridDim.x * 256;
  for (size_t i = first; i < rows * (D / 8); i += step)
    reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
  if (n_parts != nullptr)
    for (size_t i = first; i < rows; i += step) n_parts[i] = 1;
  return any;
}

}  // namespace

template <typename T, int D, bool kPaged>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_kernel(const __grid_constant__ CUtensorMap tq,
                            const __grid_constant__ CUtensorMap tk,
                            const __grid_constant__ CUtensorMap tv, PackedAttnArgs a, int tok1,
                            int n_items, int box_rows) {
  using L = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                                  // row tile X at X * kQTile
  uint8_t* k_s = q_s + 2 * L::kQTile;
  uint8_t* v_s = k_s + kStages * L::kKvTile;
  uint8_t* o_s = v_s + kStages * L::kKvTile;            // [softmax warp]
  uint64_t* bars = reinterpret_cast<uint64_t*>(o_s + 8 * L::kStage);
  uint64_t* k_full = bars;                              // [kStages]
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;                 // [2 row tiles][2 buffers]
  uint64_t* p_full = s_full + 4;
  uint64_t* pv_done = p_full + 4;
  uint64_t* o_free = pv_done + 4;                       // [2 row tiles]
  uint64_t* q_full = o_free + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* item_full = q_empty + 1;                    // [2]
  uint64_t* item_empty = item_full + 2;                 // [2]
  Item* items = reinterpret_cast<Item*>(item_empty + 2);  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = a.nq / a.nkv;
  const int block_tokens = 2 * tok1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&o_free[i], 4);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 9);  // the MMA thread and 8 softmax warps
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    // -------------------------------------------- work items, TMA producer
    auto cu_q = [&](int i) { return min(max(a.cu_q[i], 0), a.T); };
    int g = 0, qi = 0, published = 0;
    bool ok = true;
    int item = blockIdx.x;
    while (item < n_items) {
      const int unit = a.splits > 1 ? item / a.splits : item, part = item - unit * a.splits;
      const int slot = unit / a.nkv, kvh = unit % a.nkv;
      // the last sequence whose first slot is at or before `slot`; sequence
      // n_seqs stands for the rows past the last offset
      int lo = 0, hi = a.n_seqs + 1;
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + step * (lane + 1);
        const bool le = at < hi && cu_q(at) / block_tokens + at <= slot;
        const int n = __popc(__ballot_sync(0xffffffffu, le));
        hi = min(hi, lo + step * (n + 1));
        lo += step * n;
      }
      Item w;
      w.kvh = kvh;
      const int q0 = cu_q(lo), q1 = lo < a.n_seqs ? max(cu_q(lo + 1), q0) : a.T;
      const int blocks = (q1 - q0 + block_tokens - 1) / block_tokens;
      int block = blocks - 1 - (slot - (q0 / block_tokens + lo));
      if (block >= blocks) block = -1;  // a slot before the first sequence's
      int k0 = 0, len = 0;
      if (lo < a.n_seqs && block >= 0) {
        if (kPaged) {
          len = checked_len(a.seq_lens[lo], a.max_pages * a.page_size, a.status, 211);
        } else {
          const int c0 = a.cu_k[lo], c1 = a.cu_k[lo + 1];
          k0 = min(max(c0, 0), a.Tk);
          len = min(max(c1, k0), a.Tk) - k0;
          if (lane == 0 && (k0 != c0 || k0 + len != c1))
            report_status(a.status, kBoundsViolation, 212);
        }
      }
      w.row0 = q0 + block * block_tokens;
      w.tokens = q1 - w.row0;
      w.pos0 = len - (q1 - w.row0);
      const int last = len > 0 ? w.pos0 + min(w.tokens, block_tokens) - 1 : -1;
      const int steps = last >= 0 ? last / kKeys + 1 : 0;
      int first_key = 0;
      w.steps = steps;
      w.parts = 1;
      if (a.splits > 1) {
        const int parts = min(max(steps / kMinPart, 1), a.splits);
        const int first_step = steps * part / parts;
        w.steps = steps * (part + 1) / parts - first_step;
        w.parts = parts | part << 8;
        first_key = first_step * kKeys;
        w.pos0 -= first_key;
        if (part >= parts) block = -1;
      }
      if (block >= 0 && ok) {
        // hand the item to the other warps
        const int ib = published & 1;
        if (published >= 2 &&
            !__all_sync(0xffffffffu, mbar_wait(&item_empty[ib], ((published >> 1) - 1) & 1,
                                               abort_flag, a.status, 230)))
          ok = false;
        if (ok && lane == 0) {
          items[ib] = w;
          mbar_arrive(&item_full[ib]);
        }
        ++published;
        if (ok && lane == 0 && w.steps > 0) {
          if (qi > 0 && !mbar_wait(q_empty, (qi - 1) & 1, abort_flag, a.status, 231)) ok = false;
          if (ok) {
            mbar_arrive_expect_tx(q_full, 2 * L::kBoxes * G * tok1 * 128);
            for (int x = 0; x < 2; ++x)
              for (int c = 0; c < L::kBoxes; ++c)
                tma_load_3d(q_s + x * L::kQTile + c * L::kQBox, &tq, q_full, c * 64, kvh * G,
                            w.row0 + x * tok1);
            ++qi;
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        // Each lane holds the page and row of one of 32 boxes, and of one of the
        // next 32: the table's latency is off the loads' path. The copies of a
        // step go out of as many lanes at once.
        const int step_boxes = kPaged ? kKeys / box_rows : 1;  // 1, 2 or 4
        struct Box {
          int page, row;
        };
        auto look_up = [&](int box) {
          const int key = first_key + (box + lane) * box_rows;
          Box r = {0, 0};
          if (kPaged && key < len) {
            r.page = a.page_table[(size_t)lo * a.table_row + key / a.page_size];
            r.row = kvh * a.page_size + key % a.page_size;
          }
          return r;
        };
        const int my_box = lane / L::kBoxes, my_col = lane % L::kBoxes;
        Box held = look_up(0), later = look_up(32);
        for (int i = 0; i < w.steps && ok; ++i, ++g) {
          const int st = g % kStages, key0 = first_key + i * kKeys;
          const uint32_t phase = ((g / kStages) - 1) & 1;
          Box box = {kvh, k0 + key0};  // packed keys: head, first row
          if (kPaged) {
            const int first = i * step_boxes;
            if (i > 0 && first % 32 == 0) {
              held = later;
              later = look_up(first + 32);
            }
            box.page = __shfl_sync(0xffffffffu, held.page, (first + my_box) & 31);
            box.row = __shfl_sync(0xffffffffu, held.row, (first + my_box) & 31);
          }
          // rows past the sequence's end are not fetched (a box at a time)
          const int boxes = kPaged ? (min(kKeys, len - key0) + box_rows - 1) / box_rows : 1;
          if (kPaged && my_box < boxes && my_col == 0 &&
              (box.page < 0 || box.page >= a.num_pages))  // the copies fill with zeros
            report_status(a.status, kBoundsViolation, 213);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* full = kv == 0 ? &k_full[st] : &v_full[st];
            if (lane == 0) {
              if (g >= kStages && !mbar_wait(kv == 0 ? &k_empty[st] : &v_empty[st], phase,
                                             abort_flag, a.status, 232 + kv))
                ok = false;
              else
                mbar_arrive_expect_tx(full, L::kBoxes * boxes * box_rows * 128);
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            if (!ok) break;
            uint8_t* dst = (kv == 0 ? k_s : v_s) + st * L::kKvTile + my_col * L::kKvBox;
            const CUtensorMap* map = kv == 0 ? &tk : &tv;
            if (my_box < boxes) {
              if (kPaged)
                tma_load_3d(dst + my_box * box_rows * 128, map, full, my_col * 64, box.row,
                            box.page);
              else
                tma_load_3d(dst, map, full, my_col * 64, box.page, box.row);
            }
          }
        }
      }
      // the next item; with the last fetch of the launch the counter is zero again
      if (lane == 0) item = (int)gridDim.x + (int)atomicInc(
          reinterpret_cast<unsigned*>(a.counter), (unsigned)n_items - 1);
      item = __shfl_sync(0xffffffffu, item, 0);
    }
    if (ok) {
      const int ib = published & 1;
      if (published >= 2 &&
          !__all_sync(0xffffffffu, mbar_wait(&item_empty[ib], ((published >> 1) - 1) & 1,
                                             abort_flag, a.status, 234)))
        ok = false;
      if (ok && lane == 0) {
        items[ib].steps = -1;
        mbar_arrive(&item_full[ib]);
      }
    }
    if (lane == 0) {
      // every load issued must land before the CTA exits (after an abort the
      // other warps may not have waited for it)
      volatile int no_abort = 0;
      if (qi > 0) mbar_wait(q_full, (qi - 1) & 1, &no_abort, nullptr, 235, 100000000ull);
      if (!ok) {
        for (int j = max(0, g + 1 - kStages); j <= g; ++j) {
          mbar_wait(&k_full[j % kStages], (j / kStages) & 1, &no_abort, nullptr, 236, 100000000ull);
          mbar_wait(&v_full[j % kStages], (j / kStages) & 1, &no_abort, nullptr, 237, 100000000ull);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------- MMA issuer
    if (elect_one()) {
      const uint32_t idesc_s = idesc16<T>(kRows, kKeys, false);
      const uint32_t idesc_pv = idesc16<T>(kRows, D, true);
      const uint32_t q_lo = desc_lo(smem_u32(q_s), 0), k_lo = desc_lo(smem_u32(k_s), 0),
                     v_lo = desc_lo(smem_u32(v_s), L::kKvBox);
      int g = 0, it = 0, taken = 0, n = 0;
      bool ok = true;
      auto issue_s = [&](int x, int i) {
        const int idx = g + i, st = idx % kStages, buf = idx & 1;
        if (x == 0 && !mbar_wait(&k_full[st], (idx / kStages) & 1, abort_flag, a.status, 240))
          return false;
        if (idx >= 2 && !mbar_wait(&pv_done[2 * x + buf], ((idx >> 1) - 1) & 1, abort_flag,
                                   a.status, 241))
          return false;
        tc_fence_after();
        const uint32_t qa = q_lo + x * (L::kQTile >> 4), ka = k_lo + st * (L::kKvTile >> 4);
        const uint32_t d = tmem + x * 128 + buf * 64;
        umma_ss<false>(d, qa, ka, idesc_s);
#pragma unroll
        for (int kk = 1; kk < D / 16; ++kk)
          umma_ss<true>(d, qa + (((kk / 4) * L::kQBox + (kk % 4) * 32) >> 4),
                        ka + (((kk / 4) * L::kKvBox + (kk % 4) * 32) >> 4), idesc_s);
        umma_commit(&s_full[2 * x + buf]);
        if (x == 1) umma_commit(&k_empty[st]);
        if (x == 1 && i == n - 1) umma_commit(q_empty);
        return true;
      };
      auto issue_pv = [&](int x, int i) {
        const int idx = g + i, st = idx % kStages, buf = idx & 1;
        if (x == 0 && !mbar_wait(&v_full[st], (idx / kStages) & 1, abort_flag, a.status, 242))
          return false;
        if (!mbar_wait(&p_full[2 * x + buf], (idx >> 1) & 1, abort_flag, a.status, 243))
          return false;
        if (i == 0 && it > 0 && !mbar_wait(&o_free[x], (it - 1) & 1, abort_flag, a.status, 244))
          return false;
        tc_fence_after();
        const uint32_t va = v_lo + st * (L::kKvTile >> 4);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          umma_ts(tmem + 256 + x * 128, tmem + x * 128 + buf * 64 + kk * 8, va + kk * (2048 >> 4),
                  idesc_pv, kk > 0 ? 1u : (uint32_t)(i > 0));
        umma_commit(&pv_done[2 * x + buf]);
        if (x == 1) umma_commit(&v_empty[st]);
        return true;
      };
      while (ok) {
        const int ib = taken & 1;
        if (!mbar_wait(&item_full[ib], (taken >> 1) & 1, abort_flag, a.status, 245))
          break;
        n = items[ib].steps;
        mbar_arrive(&item_empty[ib]);
        ++taken;
        if (n < 0) break;
        if (n == 0) continue;
        if (!mbar_wait(q_full, it & 1, abort_flag, a.status, 246)) break;
        ok = issue_s(0, 0) && issue_s(1, 0) && (n == 1 || issue_s(0, 1));
        for (int i = 0; ok && i < n; ++i)
          ok = issue_pv(0, i) && (i + 1 >= n || issue_s(1, i + 1)) && issue_pv(1, i) &&
               (i + 2 >= n || issue_s(0, i + 2));
        g += n;
        ++it;
      }
    }
  } else {
    // ------------------------------------------- softmax, O, output rows
    const int stored_rows =  // of a tile
        settle_offsets(a.cu_q, a.n_seqs, a.T, a.nq, D, a.out, a.splits > 1 ? a.n_parts : nullptr,
                       a.status)
            ? 0
            : tok1 * G;
    const int x = (warp - 2) / 4;         // row tile of this warp group
    const int qq = warp & 3;              // TMEM lane quarter of this warp
    const int row = qq * 32 + lane;
    const int tok = x * tok1 + row / G;   // this row's token in the block
    const bool has_token = row < stored_rows;
    const int tok_first = x * tok1 + (qq * 32) / G;  // of the warp's first row
    const uint32_t lane_off = (uint32_t)(qq * 32) << 16;
    const uint32_t t_o = tmem + 256 + x * 128 + lane_off;
    const float scale_log2 = a.scale * 1.4426950408889634f;
    const float growth = fminf(8.f / scale_log2, 1e38f);
    int g = 0, taken = 0;
    bool ok = true;
    // TMEM accesses are warp-collective: every branch around them is
    // warp-uniform
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int where) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status, where));
      return ok;
    };
    while (ok) {
      const int ib = taken & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&item_full[ib], (taken >> 1) & 1, abort_flag,
                                             a.status, 250));
      if (!ok) break;
      const Item w = items[ib];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[ib]);
      ++taken;
      if (w.steps < 0) break;
      // rows past the sequence's end (never stored) see what its last row sees
      const int len = w.pos0 + w.tokens;
      const int pos = min(w.pos0 + tok, len - 1);
      const int warp_pos0 = min(w.pos0 + tok_first, len - 1);
      float top = -INFINITY;  // the running maximum, a score
      bool far = false;       // a row of the warp has a remainder in its Ref
      float2 l2 = make_float2(0.f, 0.f);
      for (int i = 0; i < w.steps; ++i, ++g) {
        const int buf = g & 1, key0 = i * kKeys;
        const uint32_t t_s = tmem + x * 128 + buf * 64 + lane_off;
        if (!wait_all(&s_full[2 * x + buf], (g >> 1) & 1, 251)) break;
        tc_fence_after();
        float s[kKeys];
        tmem_ld64(t_s, s);
        // below the diagonal for every row of this warp: nothing to mask
        if (key0 + kKeys - 1 > warp_pos0) {
#pragma unroll
          for (int k = 0; k < kKeys; ++k)
            if (key0 + k > pos) s[k] = -INFINITY;
          if (x == 0 && key0 + kKeys > len) {
            // rows past the sequence's end belong to others or to nobody: zero
            // V there, so that P = 0 meets finite values
            const int st = g % kStages;
            if (!wait_all(&v_full[st], (g / kStages) & 1, 252)) break;
            const int r = row / 2;
            if (key0 + r >= len) {
              uint8_t* vr = v_s + st * L::kKvTile + r * 128 + (row & 1) * 64;
#pragma unroll
              for (int c = 0; c < L::kBoxes; ++c)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                  *reinterpret_cast<uint4*>(vr + c * L::kKvBox + u * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int k = 4; k < kKeys - 4; k += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[k + 2 * e], s[k + 2 * e + 1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[kKeys - 4 + e]);
        const float rmax = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
        const bool grow = rmax > top + growth;
        if (__any_sync(0xffffffffu, grow)) {
          const float top_new = grow ? rmax : top;
          const Ref now = ref_of(top_new, scale_log2);
          if (i > 0) {
            // O holds steps 0 .. i-1 once P(i-1) V is done
            if (!wait_all(&pv_done[2 * x + (buf ^ 1)], ((g - 1) >> 1) & 1, 253)) break;
            tc_fence_after();
            const float alpha = grow ? exp2_approx(over(ref_of(top, scale_log2), now)) : 1.f;
            l2.x *= alpha;
            l2.y *= alpha;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              float o[16];
              tmem_ld16(t_o + c * 16, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= alpha;
              tmem_st16(t_o + c * 16, o);
            }
          }
          top = top_new;
          far = __any_sync(0xffffffffu, now.r != 0.f);
        }
        // p = 2^(s c - m); a masked s = -inf gives 0, also in a row that has seen
        // no key yet (m = -inf)
        float factor = scale_log2, neg_m = top == -INFINITY ? 0.f : -(top * scale_log2);
        if (far) {
          const float r = ref_of(top, scale_log2).r;
#pragma unroll
          for (int k = 0; k < kKeys; ++k) s[k] = fmaf(s[k], factor, neg_m) - r;
          factor = 1.f;
          neg_m = 0.f;
        }
        const float2 sc2 = make_float2(factor, factor), nm2 = make_float2(neg_m, neg_m);
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 p = fma2(make_float2(s[c * 32 + 2 * e], s[c * 32 + 2 * e + 1]), sc2, nm2);
            p.x = exp2_approx(p.x);
            p.y = exp2_approx(p.y);
            l2 = add2(l2, p);
            pk[e] = pack2<T>(p.x, p.y);
          }
          tmem_st16_raw(t_s + c * 16, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * x + buf]);
      }
      if (!ok) break;
      const float l = l2.x + l2.y;
      const float inv = 1.f / l;
      if (w.steps > 0) {
        if (!wait_all(&pv_done[2 * x + ((g - 1) & 1)], ((g - 1) >> 1) & 1, 254)) break;
        tc_fence_after();
      }
      if (a.splits > 1 && has_token && tok < w.tokens) {
        const size_t r = (size_t)(w.row0 + tok) * a.nq + w.kvh * G + row % G;
        if (w.parts < 256) a.n_parts[r] = w.parts;
        a.part_ml[(size_t)(w.parts >> 8) * a.T * a.nq + r] = make_float2(top, l);
      }
      // Through shared memory, so that a store instruction covers whole 128-byte
      // lines of four rows (a row a lane took 4100 cycles for an item's rows).
      // `Out` is the output's type, or float for a part's O as it is.
      auto store = [&](auto* base, auto kind) {
        using Out = decltype(kind);
        constexpr int kDims = 128 / sizeof(Out);
        uint8_t* stage = o_s + (warp - 2) * L::kStage;
        Out* out = reinterpret_cast<Out*>(base) +
                   ((size_t)(w.row0 + x * tok1) * a.nq + w.kvh * G) * D + lane % 8 * (kDims / 8);
#pragma unroll
        for (int c = 0; c < D / kDims; ++c) {
          float o[kDims];
          if (w.steps > 0) {
            if constexpr (kDims == 64) tmem_ld64(t_o + c * 64, o);
            else tmem_ld32(t_o + c * 32, o);
          } else {
#pragma unroll
            for (int e = 0; e < kDims; ++e) o[e] = 0.f;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            uint4 v;
            // a row that saw no key: exact zeros whatever O holds
            if constexpr (kDims == 64) {
              v.x = l == 0.f ? 0u : pack2<T>(o[8 * u + 0] * inv, o[8 * u + 1] * inv);
              v.y = l == 0.f ? 0u : pack2<T>(o[8 * u + 2] * inv, o[8 * u + 3] * inv);
              v.z = l == 0.f ? 0u : pack2<T>(o[8 * u + 4] * inv, o[8 * u + 5] * inv);
              v.w = l == 0.f ? 0u : pack2<T>(o[8 * u + 6] * inv, o[8 * u + 7] * inv);
            } else {
              v = make_uint4(__float_as_uint(o[4 * u]), __float_as_uint(o[4 * u + 1]),
                             __float_as_uint(o[4 * u + 2]), __float_as_uint(o[4 * u + 3]));
            }
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) = v;
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int rw = k * 4 + lane / 8, r = qq * 32 + rw, t = r / G;
            if (r < stored_rows && x * tok1 + t < w.tokens)
              *reinterpret_cast<uint4*>(out + ((size_t)t * a.nq + (r - t * G)) * D + c * kDims) =
                  *reinterpret_cast<const uint4*>(stage + rw * 128 +
                                                  ((lane % 8 ^ (rw & 7)) << 4));
          }
          __syncwarp();
        }
      };
      if (w.parts != 1) store(a.part_o + (size_t)(w.parts >> 8) * a.T * a.nq * D, float());
      else store(a.out, T());
      if (w.steps > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[x]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the rows that have several, D / 4 threads a row:
//   out = sum_p w_p O_p / sum_p w_p l_p,  w_p = Ref of the part / Ref of the largest
template <typename T, int D>
__global__ void __launch_bounds__(128) join_parts_kernel(PackedAttnArgs a) {
  constexpr int kLanes = D / 4;
  pdl_wait();
  pdl_trigger();
  const size_t rows = (size_t)a.T * a.nq;
  const size_t r = ((size_t)blockIdx.x * 128 + threadIdx.x) / kLanes;
  if (r >= rows) return;
  const int parts = min(a.n_parts[r], a.splits);
  if (parts <= 1) return;
  float most = -INFINITY;
  for (int p = 0; p < parts; ++p) most = fmaxf(most, a.part_ml[p * rows + r].x);
  const float scale_log2 = a.scale * 1.4426950408889634f;
  const Ref ref = ref_of(most, scale_log2);
  const int at = threadIdx.x % kLanes * 4;
  float l = 0.f, o[4] = {};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float2 ml = a.part_ml[p * rows + r];
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + (p * rows + r) * D + at);
    if (ml.y == 0.f) continue;  // the row saw none of the part's keys
    const float w = exp2_approx(over(ref_of(ml.x, scale_log2), ref));
    l = fmaf(w, ml.y, l);
    o[0] = fmaf(w, v.x, o[0]);
    o[1] = fmaf(w, v.y, o[1]);
    o[2] = fmaf(w, v.z, o[2]);
    o[3] = fmaf(w, v.w, o[3]);
  }
  const float inv = 1.f / l;
  uint2 v = make_uint2(0u, 0u);
  if (l != 0.f) v = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + r * D + at) = v;
}

// ============================================================ host side ===

int packed_attention_splits(long long T, int n_seqs, int nq, int nkv, long long most_keys,
                            int num_sms) {
  const int block = 2 * (kRows / (nq / nkv));
  const long long blocks = T / block + n_seqs / 2;  // about: a last block of each is half full
  const long long items = (blocks > 0 ? blocks : 1) * nkv;
  const long long s =
      std::min((num_sms + items / 4) / items, most_keys / (kMinPart * kKeys));
  return (int)std::min<long long>(std::max<long long>(s, 1), kMaxParts);
}

long long packed_attention_part_bytes(long long rows, int D, int splits) {
  return splits > 1 ? rows * (4 + (8 + 4ll * D) * splits) + 32 : 0;
}

template <typename T, int D, bool kPaged>
static int launch_one(const PackedAttnArgs& a, int num_sms, const CUtensorMap& tq,
                      const CUtensorMap& tk, const CUtensorMap& tv, int tok1, int box_rows,
                      cudaStream_t s) {
  const auto kern = packed_attention_kernel<T, D, kPaged>;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), Smem<D>::kBytes);
  if (e != cudaSuccess) return 4000 + (int)e;
  const long long items = ((long long)a.T / (2 * tok1) + a.n_seqs + 1) * a.nkv * a.splits;
  if (items > 0x3fffffff) return 1;
  const int grid = (int)(items < num_sms ? items : num_sms);
  e = launch_k(kern, dim3(grid), dim3(kThreads), Smem<D>::kBytes, s, tq, tk, tv, a, tok1,
               (int)items, box_rows);
  if (e == cudaSuccess && a.splits > 1) {
    const long long threads = (long long)a.T * a.nq * (D / 4);
    e = launch_k(join_parts_kernel<T, D>, dim3((unsigned)((threads + 127) / 128)), dim3(128), 0, s,
                 a);
  }
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

int launch_packed_attention(const PackedAttnArgs& a_in, void* parts, int num_sms,
                            cudaStream_t s) {
  PackedAttnArgs a = a_in;
  if (a.T == 0) return 0;
  {  // O (16-byte aligned), then (m, l), then the numbers of parts
    const long long rows = (long long)a.T * a.nq;
    if (a.splits < 1 || a.splits > kMaxParts || rows * (a.D / 4) / 128 >= 0x7fffffff) return 1;
    a.part_o = reinterpret_cast<float*>(parts);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * a.D * a.splits);
    a.n_parts = reinterpret_cast<int*>(a.part_ml + rows * a.splits);
  }
  if (!a.paged && a.Tk == 0) {  // no key anywhere
    const cudaError_t e = cudaMemsetAsync(a.out, 0, (size_t)a.T * a.nq * a.D * 2, s);
    return e == cudaSuccess ? 0 : 4000 + (int)e;
  }
  const int G = a.nq / a.nkv, tok1 = kRows / G;
  CUtensorMap tq, tk, tv;
  const uint64_t e2 = 2;  // bytes of an element
  {  // q [T, nq, D]: a box is tok1 tokens x the G heads of a kv head
    const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.nq, (uint64_t)a.T};
    const uint64_t str[2] = {a.D * e2, (uint64_t)a.q_row * e2};
    const uint32_t box[3] = {64, (uint32_t)G, (uint32_t)tok1};
    if (int e = encode_map16(&tq, a.q, a.elem, 3, dims, str, box)) return e;
  }
  int box_rows = kKeys;
  if (a.paged) {
    // pool [pages, nkv * page_size, D]: the largest box that no page ends inside
    while (a.page_size % box_rows) box_rows /= 2;
    const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.nkv * a.page_size,
                              (uint64_t)a.num_pages};
    const uint64_t str[2] = {a.D * e2, (uint64_t)a.page_stride * e2};
    const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
    if (int e = encode_map16(&tk, a.k_pages, a.elem, 3, dims, str, box)) return e;
    if (int e = encode_map16(&tv, a.v_pages, a.elem, 3, dims, str, box)) return e;
  } else {
    const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.nkv, (uint64_t)a.Tk};
    const uint32_t box[3] = {64, 1, (uint32_t)kKeys};
    const uint64_t kstr[2] = {a.D * e2, (uint64_t)a.k_row * e2};
    const uint64_t vstr[2] = {a.D * e2, (uint64_t)a.v_row * e2};
    if (int e = encode_map16(&tk, a.k, a.elem, 3, dims, kstr, box)) return e;
    if (int e = encode_map16(&tv, a.v, a.elem, 3, dims, vstr, box)) return e;
  }
#define AFD_PACKED(T, D)                                                                    \
  (a.paged ? launch_one<T, D, true>(a, num_sms, tq, tk, tv, tok1, box_rows, s)              \
           : launch_one<T, D, false>(a, num_sms, tq, tk, tv, tok1, box_rows, s))
  if (a.elem == kElemBf16)
    return a.D == 128 ? AFD_PACKED(__nv_bfloat16, 128) : AFD_PACKED(__nv_bfloat16, 64);
  return a.D == 128 ? AFD_PACKED(__half, 128) : AFD_PACKED(__half, 64);
#undef AFD_PACKED
}

}  // namespace afd
