// The whole routed-expert layer for up to 64 tokens, in one launch and without routing tables in memory.
//
//   h[e, t] = c[t, e] * SwiGLU(W13[e] x[t]),   c[t, e] = sum of the scores of token t's routes to expert e   (bf16)
//   out[t]  = sum_e W2[e] h[e, t]                                                                            (bf16)
// Products and sums are in 32 bits; h is rounded once, with the score in it, so that the second product sums over experts in its
// accumulators and has no weighted sum behind it.
//
// HBM bound: the weights of every expert that is hit stream through once (6 D F bytes each), all else is small.  So the weights never
// wait: one warp of a block brings them into a ring in shared memory (an item by one tensor copy) and goes on from W13 to W2 at once,
// another brings the rows of x or h that meet them (512 bytes by one cp.async of the warp) and alone waits for the other blocks where
// h begins: by then up to 200 KB of W2 per SM are there.  All blocks are resident at once (cooperative launch), and that wait is bounded.
//
// Measured as replayed graphs, L2 flushed, beside what the weights take at the copy rate: 64 experts x 2048 x 1408, top 6, 1 token 39 us
// (16), 4 tokens 86 (55), 32 tokens 180 (158), 64 tokens 220 (169); 32 experts x 7168 x 2048, top 8, 4 tokens 301 to 307 (295).  With
// sixteen tokens to an expert the products hold it, not the stream: 64 tokens of that layer 700 (430).  Of a call with little to read,
// 3 us go by before the first product, 1 to 2 at the meeting, and 2 to 5 on the parts of cut strips at the end.
//
// A block works on strips of 64 weight rows (32 features of gate and up; 64 output columns), 16 for each of its four warps that multiply;
// an item is 128 values of the inner dimension of a strip, 16 KiB.  A warp has its rows for itself, sums them in registers and ends a
// strip without the others: nothing but the ring's places keeps the warps together.  (With the inner dimension of an item shared by
// eight warps, the barrier and the sums in shared memory at the end of a strip stopped the stream: the 32 tokens above took 207 us.)
// Where W13 has enough strips, blocks take them by tickets; else, and for W2, the items of all strips are dealt out evenly over the
// blocks, whatever the number of experts hit.  Rows of a strip that is cut between blocks are summed by the one of the blocks' warps
// that finishes last, in the order of the blocks.
//
// With so few columns the products are mma.sync m16n8k16, weights as the 16-row operand, tokens as the 8 columns: both operands are
// then read 16 bytes a lane along the inner dimension as they lie in shared memory, its order inside 32 values being the same for both
// (lane t of a row holds values 8 t .. 8 t + 7, in two instructions), and a gate value meets its up value in the same lane.  Row g of
// the instruction is row few_row(g) of the warp's rows, which keeps the reads of the 128-byte swizzle free of bank conflicts.
#include <algorithm>
#include <type_traits>

#include "few_split.cuh"
#include "gemm_common.cuh"
#include "../../include/dist_moe_b200.h"

namespace dm {

constexpr int kFewTokens = DM_FEW_TOKENS_MAX;
constexpr int kFewExperts = 1024;
constexpr int kFewTopK = 32;
constexpr int kFewWarps = 4;                       // that multiply, 16 weight rows each
constexpr int kFewThreads = 32 * (kFewWarps + 2);  // and one that loads weights, one that loads rows of x or h
constexpr int kFewRows = 16 * kFewWarps;           // weight rows per strip
constexpr int kFewFeatures = kFewRows / 2;         // of W13
constexpr int kFewLines = 2;                       // 128-byte lines of an item's rows
constexpr int kFewStep = 64 * kFewLines;           // values of the inner dimension per item
constexpr int kFewLineBytes = kFewRows * 128;
constexpr int kFewWeightBytes = kFewLines * kFewLineBytes;  // weights of an item
constexpr int kFewRowPitch = kFewStep * 2 + 64;    // rows of x or h: eight of them, 16 bytes a lane, hit every bank once
constexpr int kFewMaxDepth = 13;
constexpr int kFewQueue = 4;                       // tickets on their way from the weights' warp to the others
__host__ __device__ constexpr int few_tiles(int T) { return T <= 8 ? 1 : T <= 16 ? 2 : T <= 32 ? 4 : 8; }
// A sum for every row and token.
__host__ __device__ constexpr int few_sum_bytes(int T) { return (kFewRows * (T | 1) * 4 + 15) / 16 * 16; }
constexpr uint64_t kFewWaitNs = 2000000000ull;

struct FewPhase {
  CUtensorMap items;  // W13 (64 values, features, gate | up, lines, experts) or W2 (64 values, columns, lines, experts)
  CUtensorMap tail;   // W2 with a last line of fewer than 64 values: (values, columns, experts)
  float* partial;     // [blocks][2][warps][tiles][32 lanes][4]
  int32_t* arrived;   // [blocks][warps], clear between calls
};
struct FewParams {
  FewPhase phase[2];  // W13, W2
  const __nv_bfloat16* x;
  const void* ids;
  const void* scores;
  int ids_are_int64, scores_are_bf16;
  __nv_bfloat16* h;  // [pairs of expert and token][F]
  __nv_bfloat16* out;
  int32_t* meeting;  // warps that have written their share of h; blocks that have seen it; tickets drawn.  Clear between calls
  int T, D, F, E, K;
  ActParams act;
  int* status;
};

// Which experts are hit, by which tokens: built by every block.
struct FewTables {
  uint2* tokens;    // [E] bit t: token t
  float* score;     // [T K]
  float* share;     // [pairs] c[t, e]
  int16_t* expert;  // [active]
  int16_t* base;    // [active + 1] first pair
  int16_t* first;   // [E] the same by expert
  int16_t* id;      // [T K]
  uint8_t* token;   // [pairs]
  __device__ __forceinline__ FewTables(uint8_t* at, int T, int E, int K) {
    const int active = T * K < E ? T * K : E;
    tokens = reinterpret_cast<uint2*>(at);
    score = reinterpret_cast<float*>(tokens + E);
    share = score + T * K;
    expert = reinterpret_cast<int16_t*>(share + T * K);
    base = expert + active;
    first = base + active + 1;
    id = first + E;
    token = reinterpret_cast<uint8_t*>(id + T * K);
  }
  static __host__ __device__ constexpr int bytes(int T, int E, int K) {
    return (10 * E + 11 * T * K + 4 * (T * K < E ? T * K : E) + 2 + 15) / 16 * 16;
  }
};

__device__ __forceinline__ int few_id(const FewParams& p, int i) {
  if (p.ids_are_int64) {
    const int64_t v = static_cast<const int64_t*>(p.ids)[i];
    return v >= 0 && v < p.E ? static_cast<int>(v) : v == -1 ? -1 : -2;
  }
  const int v = static_cast<const int32_t*>(p.ids)[i];
  return v >= 0 && v < p.E ? v : v == -1 ? -1 : -2;
}

__device__ __forceinline__ float few_score(const FewParams& p, int i) {
  return p.scores_are_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.scores)[i]) : static_cast<const float*>(p.scores)[i];
}

// All warps: the experts that are hit and their pairs' places.  Returns their number; `most` is the largest number of tokens of one.
__device__ __forceinline__ int few_tables(const FewParams& p, const FewTables& s, int (&s_found)[2], bool report, int& most) {
  const int routes = p.T * p.K;
  int i = threadIdx.x, id = -1;
  float score = 0.f;
  if (i < routes) {  // on their way while the masks are cleared
    id = few_id(p, i);
    score = few_score(p, i);
  }
  for (int e = threadIdx.x; e < p.E; e += kFewThreads) s.tokens[e] = make_uint2(0, 0);
  __syncthreads();
  while (i < routes) {
    const int t = i / p.K;
    s.score[i] = score;
    s.id[i] = static_cast<int16_t>(id);
    if (id >= 0)
      atomicOr(t < 32 ? &s.tokens[id].x : &s.tokens[id].y, 1u << (t & 31));
    else if (id == -2 && report)
      set_status(p.status, kInvalidExpertId, i);
    i += kFewThreads;
    if (i < routes) {
      id = few_id(p, i);
      score = few_score(p, i);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int active = 0, pairs = 0, largest = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const uint2 tokens = e0 + lane < p.E ? s.tokens[e0 + lane] : make_uint2(0, 0);
      const int own = __popc(tokens.x) + __popc(tokens.y);
      const uint32_t hit = __ballot_sync(0xffffffffu, own != 0);
      int before = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += v;
      }
      const int total = __shfl_sync(0xffffffffu, before, 31);
      if (own != 0) {
        const int at = active + __popc(hit & ((1u << lane) - 1)), n = pairs + before - own;
        s.expert[at] = static_cast<int16_t>(e0 + lane);
        s.base[at] = s.first[e0 + lane] = static_cast<int16_t>(n);
      }
      active += __popc(hit);
      pairs += total;
      largest = max(largest, own);
    }
    largest = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<uint32_t>(largest)));
    if (lane == 0) {
      s.base[active] = static_cast<int16_t>(pairs);
      s_found[0] = active;
      s_found[1] = largest;
    }
  }
  __syncthreads();
  most = s_found[1];
  return s_found[0];
}

// The warps that need them, thread `rank` of `ranks`: the pairs' tokens and shares, a pair by the first of its routes.
__device__ __forceinline__ void few_pairs(const FewParams& p, const FewTables& s, int rank, int ranks) {
  for (int i = rank; i < p.T * p.K; i += ranks) {
    const int id = s.id[i], t = i / p.K, row = t * p.K;
    if (id < 0) continue;
    bool again = false;
    float share = 0.f;
    for (int j = row; j < row + p.K; ++j) {
      const bool same = s.id[j] == id;
      again = again || (same && j < i);
      if (same) share += s.score[j];
    }
    if (again) continue;
    const uint2 tokens = s.tokens[id];
    const uint32_t below = (1u << (t & 31)) - 1;
    const int pair = s.first[id] + (t < 32 ? __popc(tokens.x & below) : __popc(tokens.x) + __popc(tokens.y & below));
    s.token[pair] = static_cast<uint8_t>(t);
    s.share[pair] = share;
  }
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* tmap, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const void* tmap, int c0, int c1, int c2, int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// Arrives once the copies of this thread so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Row g of the instruction: neighbouring ones differ in the swizzle's third bit.
__device__ __forceinline__ constexpr int few_row(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ int atom_add_acq_rel(int32_t* p, int v) {
  int old;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// Where a block stands: strip, active expert, step of the inner dimension.  W13: strips of an expert follow one another; W2: the
// experts of a strip do, and are summed.
template <bool kDown>
struct FewCursor {
  int strip, a, c;
  __device__ __forceinline__ void set(uint32_t item, uint32_t strips, uint32_t active, uint32_t steps) {
    const uint32_t rest = item / steps, of = kDown ? active : strips, outer = rest / of;
    c = item - rest * steps;
    (kDown ? a : strip) = rest - outer * of;
    (kDown ? strip : a) = outer;
  }
  __device__ __forceinline__ void next(int strips, int active, int steps) {
    if (++c < steps) return;
    c = 0;
    if (kDown) {
      if (++a < active) return;
      a = 0;
      ++strip;
    } else {
      if (++strip < strips) return;
      strip = 0;
      ++a;
    }
  }
};

// Whole strips by tickets, where the rounds are three quarters full or more on average: nothing is cut then, and blocks that are served
// faster take more.  Even shares took 2 to 5 % longer from 0.74 full up in 2 to 5 rounds, 10 % in 10 and more (32 tokens of 64 experts x
// 2048 x 1408 199 us against 181, 4 of 32 x 7168 x 2048 336 against 307); tickets took 3 % longer at 0.72 and 9 % at 0.65 (5 and 3
// experts x 7168 x 2048).
__device__ __forceinline__ bool few_by_tickets(uint32_t strips, uint32_t blocks) {
  const uint64_t rounds = (strips + blocks - 1) / blocks;
  return 4ull * strips >= 3 * rounds * blocks;
}

// What the warps of a block know of one of the two products.
template <bool kDown>
struct FewWork {
  int inner, steps, strips, length, items;
  FewSplit split;
  FewCursor<kDown> begin;
  bool tickets;  // strips are drawn one after another, the first one by the block's number; else the block has one run of items
  __device__ __forceinline__ FewWork(const FewParams& p, int active)
      : inner(kDown ? p.F : p.D),
        steps((inner + kFewStep - 1) / kFewStep),
        strips(kDown ? p.D / kFewRows : (p.F + kFewFeatures - 1) / kFewFeatures),  // W13: of one expert
        length(kDown ? active * steps : steps),            // items of a strip
        split(kDown ? strips : active * strips, length, gridDim.x) {
    const uint32_t first = split.begin(blockIdx.x);
    items = split.end(blockIdx.x) - first;
    begin.set(0, 1, 1, 1);
    tickets = !kDown && few_by_tickets(active * strips, gridDim.x);
    if (tickets)
      draw(blockIdx.x, active);
    else if (items > 0)
      begin.set(first, strips, active, steps);
  }
  // The strip of a ticket; no items behind the last one.
  __device__ __forceinline__ void draw(int ticket, int active) {
    items = ticket < active * strips ? steps : 0;
    if (items > 0) begin.set(ticket * steps, strips, active, steps);
  }
};

struct FewQueue {
  uint64_t* full;
  uint64_t* empty;
  int* ticket;
  int n;  // tickets seen
  __device__ __forceinline__ int place() const { return n & (kFewQueue - 1); }
  __device__ __forceinline__ uint32_t round() const { return (n / kFewQueue) & 1; }
  // The next ticket, for a whole warp; -1 if it did not come in time.
  __device__ __forceinline__ int next(int* abort_flag, int lane) {
    if (!warp_mbar_wait(&full[place()], round(), abort_flag)) return -1;
    const int got = ticket[place()];
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[place()]);
    ++n;
    return got;
  }
};

struct FewRing {
  uint8_t* base;
  uint64_t* full;
  uint64_t* empty;
  int* abort_flag;
  int place_bytes, depth;
  int place;
  uint32_t round;  // parity of the ring's round
  __device__ __forceinline__ void next() {
    if (++place == depth) {
      place = 0;
      round ^= 1u;
    }
  }
};

// The weights' warp, all lanes.  Returns whether every place became free in time.
template <bool kDown>
__device__ __forceinline__ bool few_load_weights(const FewParams& p, const FewTables& tab, FewRing& ring, FewQueue& queue, int active, bool elected,
                                                 int lane) {
  FewWork<kDown> work(p, active);
  const FewPhase& phase = p.phase[kDown];
  while (true) {
    int next = 0;
    if (work.tickets && work.items > 0 && lane == 0) next = gridDim.x + atomicAdd(p.meeting + 2, 1);  // here by the end of this strip
    FewCursor<kDown> at = work.begin;
    for (int i = 0; i < work.items; ++i) {
      if (!warp_mbar_wait(&ring.empty[ring.place], ring.round ^ 1u, ring.abort_flag)) return false;
      uint8_t* to = ring.base + ring.place * ring.place_bytes;
      uint64_t* full = &ring.full[ring.place];
      const int e = uniform(static_cast<int>(tab.expert[at.a])), strip = uniform(at.strip), c = uniform(at.c);
      if (elected) {
        if (kDown && (c + 1) * kFewStep > work.inner && (work.inner & 63) != 0) {
          const int lines = min(kFewLines, (work.inner - c * kFewStep + 63) / 64);
          mbar_arrive_expect_tx(full, lines * kFewLineBytes);
          for (int l = 0; l < lines; ++l)
            tma_load_3d(to + l * kFewLineBytes, &phase.tail, c * kFewStep + 64 * l, strip * kFewRows, e, full);
        } else {
          mbar_arrive_expect_tx(full, kFewWeightBytes);
          if (kDown)
            tma_load_4d(to, &phase.items, 0, strip * kFewRows, c * kFewLines, e, full);
          else
            tma_load_5d(to, &phase.items, 0, strip * kFewFeatures, 0, c * kFewLines, e, full);
        }
      }
      __syncwarp();
      at.next(work.strips, active, work.steps);
      ring.next();
    }
    if (!work.tickets || work.items == 0) return true;
    next = uniform(next);
    if (!warp_mbar_wait(&queue.empty[queue.place()], queue.round() ^ 1u, ring.abort_flag)) return false;
    if (lane == 0) {
      queue.ticket[queue.place()] = next;
      mbar_arrive(&queue.full[queue.place()]);
    }
    __syncwarp();
    ++queue.n;
    work.draw(next, active);
  }
}

// The rows' warp, all lanes: the expert's rows next to one another.
template <bool kDown>
__device__ __forceinline__ bool few_load_rows(const FewParams& p, const FewTables& tab, FewRing& ring, FewQueue& queue, int active, int lane) {
  FewWork<kDown> work(p, active);
  const int piece = lane & 15, first = lane >> 4;  // 16 lanes a row
  const uint32_t own = smem_u32(ring.base) + kFewWeightBytes + piece * 16;
  while (true) {
    FewCursor<kDown> at = work.begin;
    for (int i = 0; i < work.items; ++i) {
      if (!warp_mbar_wait(&ring.empty[ring.place], ring.round ^ 1u, ring.abort_flag)) return false;
      const int k = at.c * kFewStep + piece * 8;
      const bool in = k < work.inner;
      const int base = tab.base[at.a], count = tab.base[at.a + 1] - base;
      const __nv_bfloat16* source = (kDown ? p.h + static_cast<int64_t>(base) * work.inner : p.x) + (in ? k : 0);
      const uint32_t to = own + ring.place * ring.place_bytes;
#pragma unroll 4
      for (int j = first; j < count; j += 2)
        cp_async16(to + j * kFewRowPitch, source + static_cast<int64_t>(kDown ? j : tab.token[base + j]) * work.inner, in);
      cp_async_arrive(&ring.full[ring.place]);
      at.next(work.strips, active, work.steps);
      ring.next();
    }
    if (!work.tickets || work.items == 0) return true;
    const int next = queue.next(ring.abort_flag, lane);
    if (next < 0) return false;
    work.draw(next, active);
  }
}

__device__ __forceinline__ bool try_wait_addr(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ void arrive_addr(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A wait that ran out is recorded; the block goes on without its data, so that its warps still meet.
__device__ __noinline__ void few_wait_on(uint64_t* bar, uint32_t parity, int* abort_flag, int* status) {
  if (!mbar_wait(bar, parity, abort_flag)) set_status(status, kPipelineTimeout, 7, blockIdx.x);
}

// The warps that multiply.  kTiles: tiles of eight columns that the accumulators hold.  Columns are an expert's tokens, next to one
// another.  At the end of a strip the sums go through shared memory; W2, which sums over the experts, adds them there by token after each
// expert.  (With all tokens as W2's columns, zero where they are not the expert's, 32 and 64 tokens of the layer above took 15 and 85 us
// more, and a weight that is not finite reached every token.)  What the warps run has to stay small: most of it runs a few times only,
// from instruction memory, and every tile's activation or partial sums written out in a row made the launch slower.
template <bool kDown, int kTiles>
__device__ __forceinline__ void few_multiply(const FewParams& p, const FewTables& tab, FewRing& ring, FewQueue& queue, int active, float* all_sums) {
  FewWork<kDown> work(p, active);
  const FewPhase& phase = p.phase[kDown];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, quad = lane & 3;
  const int rho = few_row(g);
  // Rows of the lane: r0 and r0 + up.  W13: the first half of a strip's rows are gate features, the second the same features of up.
  constexpr int up = kDown ? 8 : kFewFeatures;
  const int r0 = warp * (kDown ? 16 : 8) + rho;
  const uint32_t at_w = smem_u32(ring.base) + r0 * 128 + ((quad ^ rho) << 4);
  const uint32_t at_b = smem_u32(ring.base) + kFewWeightBytes + quad * 16;
  const uint32_t full0 = smem_u32(ring.full), empty0 = smem_u32(ring.empty);
  int place = ring.place;
  uint32_t round = ring.round, here = place * ring.place_bytes;
  float acc[kTiles][4];
  auto clear = [&] {
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
  };
  const int pitch = p.T | 1;
  float* sums = all_sums + warp * 16 * pitch;  // of this warp's rows, by token
  auto clear_sums = [&] {
    for (int i = lane; i < 16 * pitch; i += 32) sums[i] = 0.f;
    __syncwarp();
  };
  int tiles = 0;
  int from[kTiles];  // offset of the column's row in a place
  auto columns = [&](int a) {  // columns beyond the last token repeat it, and are not kept
    const int count = tab.base[a + 1] - tab.base[a];
    tiles = (count + 7) >> 3;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) from[n] = min(8 * n + g, count - 1) * kFewRowPitch;
  };
  // A line's operands.
  struct Operands {
    uint4 lo[2], hi[2], b[2];
  };
  auto wait = [&] {
    if (!try_wait_addr(full0 + 8 * place, round)) few_wait_on(ring.full + place, round, ring.abort_flag, p.status);
  };
  auto fetch = [&](Operands& x, int line) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t aw = (at_w + here + line * kFewLineBytes) ^ (h << 6);
      x.lo[h] = lds16(aw);
      x.hi[h] = lds16(aw + up * 128);
      x.b[h] = lds16(at_b + here + from[0] + line * 128 + h * 64);
    }
  };
  // 32 values are two instructions.  An instruction waits for the one before it on the same accumulators, and a warp issues in order:
  // others stand between the two.
  auto first_half = [&](float (&to)[4], const Operands& x, const uint4& b, int h) {
    mma_16x8x16(to, x.lo[h].x, x.hi[h].x, x.lo[h].y, x.hi[h].y, b.x, b.y);
  };
  auto second_half = [&](float (&to)[4], const Operands& x, const uint4& b, int h) {
    mma_16x8x16(to, x.lo[h].z, x.hi[h].z, x.lo[h].w, x.hi[h].w, b.z, b.w);
  };
  auto leave = [&] {  // the item's place is read
    __syncwarp();
    if (lane == 0) arrive_addr(empty0 + 8 * place);
    ++place;
    here += ring.place_bytes;
    if (place == ring.depth) {
      place = 0;
      here = 0;
      round ^= 1u;
    }
  };
  // `n_items` items in a row with `lines` lines of values.  Beyond them a place holds anything; in the last one zeros follow the values.
  auto run_one_tile = [&](int n_items, int lines) {
    float more[3][4] = {};
    Operands x, y;
#pragma unroll 1
    for (int i = 0; i < n_items; ++i, lines -= kFewLines) {
      wait();
      fetch(x, 0);
      if (lines > 1) fetch(y, 1);
      leave();
      first_half(acc[0], x, x.b[0], 0);
      first_half(more[0], x, x.b[1], 1);
      if (lines > 1) {
        first_half(more[1], y, y.b[0], 0);
        first_half(more[2], y, y.b[1], 1);
      }
      second_half(acc[0], x, x.b[0], 0);
      second_half(more[0], x, x.b[1], 1);
      if (lines > 1) {
        second_half(more[1], y, y.b[0], 0);
        second_half(more[2], y, y.b[1], 1);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[0][j] += more[0][j] + (more[1][j] + more[2][j]);
  };
  auto run = [&](int n_items, int lines) {
    float more[kTiles][4] = {};  // for every second 32 values
    Operands x, y;
    uint4 b[2][4];
    auto load = [&](uint4 (&to)[4], int n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = lds16(at_b + here + from[n] + i * 64);
    };
#pragma unroll 1
    for (int i = 0; i < n_items; ++i, lines -= kFewLines) {
      wait();
      fetch(x, 0);
      fetch(y, 1);
      if (lines <= 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) y.lo[h] = y.hi[h] = make_uint4(0, 0, 0, 0);
      }
      b[0][0] = x.b[0], b[0][1] = x.b[1], b[0][2] = y.b[0], b[0][3] = y.b[1];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        if (n >= tiles) break;
        const uint4(&now)[4] = b[n & 1];
        if (n + 1 < kTiles) load(b[(n + 1) & 1], n + 1);
        first_half(acc[n], x, now[0], 0);
        first_half(more[n], x, now[1], 1);
        second_half(acc[n], x, now[0], 0);
        second_half(more[n], x, now[1], 1);
        first_half(acc[n], y, now[2], 0);
        first_half(more[n], y, now[3], 1);
        second_half(acc[n], y, now[2], 0);
        second_half(more[n], y, now[3], 1);
      }
      leave();
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] += more[n][j];
  };
  clear();
  if (kDown) clear_sums();
  FewCursor<kDown> at = work.begin;
  bool whole = at.c == 0 && (!kDown || at.a == 0);  // the strip from its first item on
  for (int left = work.items; left > 0;) {
    columns(at.a);
    const int n_items = min(left, work.steps - at.c);
    const int lines = (work.inner - at.c * kFewStep + 63) / 64;
    if (kTiles == 1 || tiles == 1)
      run_one_tile(n_items, lines);
    else
      run(n_items, lines);
    left -= n_items;
    const FewCursor<kDown> done = at;
    const int base = tab.base[at.a], pairs = tab.base[at.a + 1] - base;
    at.c += n_items - 1;
    at.next(work.strips, active, work.steps);
    const bool strip_end = kDown ? at.strip != done.strip : at.c == 0;
    const bool ends = strip_end || left == 0;
    if (kDown || ends) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        if (n >= tiles) break;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int col = 8 * n + 2 * quad + j;
          if (col < pairs) {
            float* to = sums + (kDown ? tab.token[base + col] : col) + rho * pitch;
            to[0] = kDown ? to[0] + acc[n][j] : acc[n][j];
            to[8 * pitch] = kDown ? to[8 * pitch] + acc[n][2 + j] : acc[n][2 + j];
          }
        }
      }
      __syncwarp();
      clear();
    }
    if (!ends) continue;
    // ---- the end of the strip, or of the block's part of it ------------------------------------------------------------------
    const int cols = kDown ? p.T : pairs;
    bool mine = true;  // to finish these rows
    if (!(whole && strip_end)) {
      // What the warps with the same rows do in every block: store their parts, arrive, and the last one finds all parts.
      const int q = kDown ? done.strip : done.a * work.strips + done.strip;  // strip of the product
      const int first = work.split.first_block(q), last = work.split.last_block(q);
      // The block that a strip begins in keeps it in the second of its places, unless it begins with it; all others in the first.
      constexpr int kPart = kFewWarps * kTiles * 32;
      float4* parts = reinterpret_cast<float4*>(phase.partial) + warp * kTiles * 32 + lane;
      const int first_place = work.split.place(first, q);
      auto part = [&](int block) { return parts + (block == first ? first_place : 2 * block) * kPart; };
      // A lane's pieces: its row, four columns after another.
      float* row = sums + (lane & 15) * pitch;
      const int col0 = 4 * (lane >> 4), used = (cols + 7) >> 3;
#pragma unroll 1
      for (int n = 0; n < used; ++n) {
        const int c = 8 * n + col0;
        __stcg(part(blockIdx.x) + n * 32, make_float4(c < cols ? row[c] : 0.f, c + 1 < cols ? row[c + 1] : 0.f, c + 2 < cols ? row[c + 2] : 0.f,
                                                     c + 3 < cols ? row[c + 3] : 0.f));
      }
      __syncwarp();
      int before = 0;
      if (lane == 0) {
        int32_t* arrived = phase.arrived + first * kFewWarps + warp;
        before = atom_add_acq_rel(arrived, 1);
        if (before == last - first) *arrived = 0;  // clear for the next call
      }
      mine = __shfl_sync(0xffffffffu, before, 0) == last - first;
      __syncwarp();  // what lane 0 acquired the other lanes read: a shuffle does not order memory
      if (mine) {
#pragma unroll 1
        for (int n0 = 0; n0 < used; n0 += 4) {
          // Up to four pieces of four blocks on their way at a time; they are summed in the blocks' order.
          constexpr int kN = kTiles < 4 ? kTiles : 4, kBlocks = 4;
          float4 v[kN];
#pragma unroll
          for (int i = 0; i < kN; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
          for (int block = first; block <= last; block += kBlocks) {
            float4 add[kBlocks][kN];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              const float4* theirs = part(block + b) + n0 * 32;
#pragma unroll
              for (int i = 0; i < kN; ++i)  // beyond `used` a place holds anything
                add[b][i] = block + b <= last ? __ldcg(theirs + i * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
              for (int i = 0; i < kN; ++i) v[i].x += add[b][i].x, v[i].y += add[b][i].y, v[i].z += add[b][i].z, v[i].w += add[b][i].w;
          }
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const int c = 8 * (n0 + i) + col0;
            if (c < cols) row[c] = v[i].x;
            if (c + 1 < cols) row[c + 1] = v[i].y;
            if (c + 2 < cols) row[c + 2] = v[i].z;
            if (c + 3 < cols) row[c + 3] = v[i].w;
          }
        }
        __syncwarp();
      }
    }
    if (mine) {
      if (kDown) {
        // two columns of four tokens at a time
        const float* row = sums + 2 * (lane & 7) * pitch;
        __nv_bfloat16* to = p.out + done.strip * kFewRows + warp * 16 + 2 * (lane & 7);
#pragma unroll 2
        for (int t = lane >> 3; t < p.T; t += 4)
          *reinterpret_cast<uint32_t*>(to + static_cast<int64_t>(t) * p.D) = pack_bf16x2(row[t], row[pitch + t]);
      } else {  // eight features of four pairs at a time
        const int f = done.strip * kFewFeatures + warp * 8 + (lane & 7);
        const float* row = sums + (lane & 7) * pitch;
        if (f < p.F)
#pragma unroll 1
          for (int col = lane >> 3; col < pairs; col += 4) {
            const float gate[1] = {row[col]}, up1[1] = {row[8 * pitch + col]};
            float z[1];
            swiglu_f32(gate, up1, z, p.act);
            p.h[static_cast<int64_t>(base + col) * p.F + f] = __float2bfloat16_rn(tab.share[base + col] * z[0]);
          }
      }
    }
    __syncwarp();
    if (kDown) clear_sums();
    whole = true;
    if (work.tickets) {
      const int next = queue.next(ring.abort_flag, lane);
      work.draw(next < 0 ? 0x7fffffff : next, active);
      at = work.begin;
      left = work.items;
    }
  }
  ring.place = place;
  ring.round = round;
}

template <int kTiles>
__global__ void __launch_bounds__(kFewThreads, 1) few_tokens_kernel(const __grid_constant__ FewParams p, int ring_bytes) {
  extern __shared__ __align__(1024) uint8_t few_smem_raw[];
  uint8_t* smem = few_smem_raw + (-smem_u32(few_smem_raw) & 1023u);  // an offset: what lies there stays known as shared memory
  __shared__ uint64_t full[kFewMaxDepth], empty[kFewMaxDepth], queue_full[kFewQueue], queue_empty[kFewQueue];
  __shared__ int s_found[2], s_ticket[kFewQueue], abort_flag;
  float* sums = reinterpret_cast<float*>(smem + ring_bytes);
  const FewTables tab(smem + ring_bytes + few_sum_bytes(p.T), p.T, p.E, p.K);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == kFewWarps) {
    if (lane < kFewMaxDepth) {
      mbar_init(&full[lane], 1 + 32);  // the weights' warp and every lane of the rows' warp
      mbar_init(&empty[lane], kFewWarps);
    }
    if (lane < kFewQueue) {
      mbar_init(&queue_full[lane], 1);
      mbar_init(&queue_empty[lane], 1 + kFewWarps);  // the rows' warp and those that multiply
    }
    if (lane == 0) {
      abort_flag = 0;
      tma_prefetch_desc(&p.phase[0].items);
      if (p.F >= 64) tma_prefetch_desc(&p.phase[1].items);
    }
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  int most;
  const int active = few_tables(p, tab, s_found, blockIdx.x == 0, most);
  if (active == 0) {  // nothing is routed anywhere: all blocks see it
    const int64_t n = static_cast<int64_t>(p.T) * p.D;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kFewThreads) + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kFewThreads)
      p.out[i] = __float2bfloat16_rn(0.f);
    return;
  }
  // A place of the ring: 16 KiB of weights, and as many rows of x or h as the expert with the most tokens has.
  FewRing ring{smem, full, empty, &abort_flag, kFewWeightBytes + (most * kFewRowPitch + 1023) / 1024 * 1024, 0, 0, 0};
  ring.depth = min(kFewMaxDepth, ring_bytes / ring.place_bytes);
  FewQueue queue{queue_full, queue_empty, s_ticket, 0};

  if (warp == kFewWarps) {
    const bool elected = elect_one();
    const bool ok = few_load_weights<false>(p, tab, ring, queue, active, elected, lane) &&
                    few_load_weights<true>(p, tab, ring, queue, active, elected, lane);
    if (lane == 0) {  // what is on its way has to land before the block gives its shared memory back
      if (!ok) set_status(p.status, kPipelineTimeout, 6, blockIdx.x);
      settle_ring(full, ring.depth, ring_stop(ring.place, ring.round), globaltimer_ns() + (ok ? kFewWaitNs : kSettleNs));
    }
    return;
  }
  constexpr int kOthers = 32 * (kFewWarps + 1);
  few_pairs(p, tab, warp == kFewWarps + 1 ? 32 * kFewWarps + lane : threadIdx.x, kOthers);
  asm volatile("bar.sync 1, %0;" ::"n"(kOthers) : "memory");
  if (warp == kFewWarps + 1) {
    bool ok = few_load_rows<false>(p, tab, ring, queue, active, lane);
    if (ok) {  // until h is there
      const uint64_t t0 = globaltimer_ns();
      uint32_t spins = 0;
      while (ok && ld_acquire_gpu(p.meeting) < static_cast<int>(gridDim.x) * kFewWarps)
        if ((++spins & 0xff) == 0 && (*const_cast<volatile int*>(&abort_flag) != 0 || globaltimer_ns() - t0 > kFewWaitNs)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      // the last one to leave clears them for the next call: every block has drawn its last ticket
      if (ok && lane == 0 && atom_add_acq_rel(p.meeting + 1, 1) == static_cast<int>(gridDim.x) - 1) p.meeting[0] = p.meeting[1] = p.meeting[2] = 0;
      __syncwarp();
    }
    ok = ok && few_load_rows<true>(p, tab, ring, queue, active, lane);
    if (!ok && lane == 0) {
      *const_cast<volatile int*>(&abort_flag) = 1;
      set_status(p.status, kPipelineTimeout, 8, blockIdx.x);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    few_multiply<false, kTiles>(p, tab, ring, queue, active, sums);
    __syncwarp();  // the warp's share of h is written
    if (lane == 0) red_release_gpu_add(p.meeting, 1);
    few_multiply<true, kTiles>(p, tab, ring, queue, active, sums);
  }
}

// An item of W13: (64 values, 32 features, gate and up, two lines); of W2: (64 values, 64 columns, two lines).  Beyond the last line or
// feature a box holds zeros.  `tail`: a line of W2 at a time, zeros beyond the last value.
static int few_encode(CUtensorMap* tm, const void* w, int64_t D, int64_t F, int64_t E, bool down, bool tail) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return kRcNoDriver;
  const cuuint64_t d = static_cast<cuuint64_t>(D), f = static_cast<cuuint64_t>(F), e = static_cast<cuuint64_t>(E);
  const cuuint64_t dims13[5] = {64, f, 2, d / 64, e}, strides13[4] = {2 * d, 2 * f * d, 128, 4 * f * d};
  const cuuint64_t dims2[4] = {64, d, f / 64, e}, strides2[3] = {2 * f, 128, 2 * f * d};
  const cuuint64_t dims_tail[3] = {f, d, e}, strides_tail[2] = {2 * f, 2 * f * d};
  const cuuint32_t box13[5] = {64, kFewFeatures, 2, kFewLines, 1}, box2[4] = {64, kFewRows, kFewLines, 1}, box_tail[3] = {64, kFewRows, 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, tail ? 3 : down ? 4 : 5, const_cast<void*>(w),
                         tail ? dims_tail : down ? dims2 : dims13, tail ? strides_tail : down ? strides2 : strides13,
                         tail ? box_tail : down ? box2 : box13, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? kRcOk : 1000 + static_cast<int>(r);
}

struct FewLayout {
  int64_t meeting, arrived13, arrived2, partial13, partial2, h, total;
};
static FewLayout few_layout(int64_t T, int64_t F, int64_t K) {
  auto a128 = [](int64_t v) { return (v + 127) / 128 * 128; };
  const int64_t blocks = sm_count(), tiles = few_tiles(static_cast<int>(T));
  const int64_t partial = a128(blocks * 2 * kFewRows * 8 * tiles * 4), arrived = a128(blocks * kFewWarps * 4);
  FewLayout l;
  l.meeting = 0;
  l.arrived13 = 128;
  l.arrived2 = l.arrived13 + arrived;
  l.partial13 = std::max<int64_t>(l.arrived2 + arrived, DM_FEW_TOKENS_COUNTER_BYTES);
  l.partial2 = l.partial13 + partial;
  l.h = l.partial2 + partial;
  l.total = l.h + a128(T * K * F * 2);
  return l;
}
static int few_shape(int64_t T, int64_t D, int64_t F, int64_t E, int64_t K) {
  if (T <= 0 || D <= 0 || F <= 0 || E <= 0 || K <= 0) return kRcBadArg;
  if (T > kFewTokens || E > kFewExperts || K > kFewTopK) return kRcTooLarge;
  if (D % 64 != 0 || F % 8 != 0 || 128 + 2 * (sm_count() * kFewWarps * 4 + 127) > DM_FEW_TOKENS_COUNTER_BYTES) return kRcUnsupportedShape;
  const int64_t active = T * K < E ? T * K : E, most = int64_t{1} << 30;  // items, counted in 32 bits
  if (D > most || F > most || ceil_div64(F, kFewFeatures) * ceil_div64(D, kFewStep) > most / active ||
      D / kFewRows * ceil_div64(F, kFewStep) > most / active)
    return kRcTooLarge;
  return kRcOk;
}

}  // namespace dm

using namespace dm;

extern "C" int64_t dm_few_tokens_workspace_bytes(int64_t T, int64_t D, int64_t F, int E, int K) {
  const int rc = few_shape(T, D, F, E, K);
  return rc != kRcOk ? rc : few_layout(T, F, K).total;
}

extern "C" int dm_few_tokens(const void* x, const void* ids, int ids_are_int64, const void* scores, int scores_are_bf16,
                             const void* w13, const void* w2, void* out, int64_t T, int64_t D, int64_t F, int E, int K, int clamped,
                             float alpha, float limit, void* workspace, int64_t workspace_bytes, int num_sms, int* status,
                             void* stream) {
  if (!x || !ids || !scores || !w13 || !w2 || !out || !workspace) return kRcBadArg;
  int rc = few_shape(T, D, F, E, K);
  if (rc != kRcOk) return rc;
  for (const void* v : {x, w13, w2, static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(v) % 16 != 0) return kRcBadArg;
  const FewLayout l = few_layout(T, F, K);
  if (workspace_bytes < l.total) return kRcBadArg;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  FewParams p{};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.ids = ids;
  p.scores = scores;
  p.ids_are_int64 = ids_are_int64;
  p.scores_are_bf16 = scores_are_bf16;
  p.h = reinterpret_cast<__nv_bfloat16*>(ws + l.h);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.meeting = reinterpret_cast<int32_t*>(ws + l.meeting);
  p.T = static_cast<int>(T), p.D = static_cast<int>(D), p.F = static_cast<int>(F), p.E = E, p.K = K;
  p.act = ActParams{clamped, alpha, limit};
  p.status = status;
  p.phase[0].partial = reinterpret_cast<float*>(ws + l.partial13);
  p.phase[0].arrived = reinterpret_cast<int32_t*>(ws + l.arrived13);
  p.phase[1].partial = reinterpret_cast<float*>(ws + l.partial2);
  p.phase[1].arrived = reinterpret_cast<int32_t*>(ws + l.arrived2);
  rc = few_encode(&p.phase[0].items, w13, D, F, E, false, false);
  if (rc == kRcOk && F >= 64) rc = few_encode(&p.phase[1].items, w2, D, F, E, true, false);
  if (rc == kRcOk && F % 64 != 0) rc = few_encode(&p.phase[1].tail, w2, D, F, E, true, true);
  if (rc != kRcOk) return rc;
  auto run = [&](auto tiles_tag) {
    constexpr auto kernel = few_tokens_kernel<decltype(tiles_tag)::value>;
    constexpr int most = 226 * 1024;
    const int red = few_sum_bytes(p.T), tables = FewTables::bytes(p.T, p.E, p.K);
    const int ring = (most - 1024 - red - tables) / 1024 * 1024;
    static PerDeviceOnce attr_set;
    const int arc = once_per_device(attr_set, [] {
      return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    });
    if (arc != 0) return arc;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeCooperative;  // the blocks meet once: all of them are resident
    attr.val.cooperative = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(persistent_grid(num_sms)));
    config.blockDim = dim3(kFewThreads);
    config.dynamicSmemBytes = 1024 + ring + red + tables;
    config.stream = static_cast<cudaStream_t>(stream);
    config.attrs = &attr;
    config.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, p, ring));
  };
  using std::integral_constant;
  if (T <= 8) return run(integral_constant<int, 1>{});
  if (T <= 16) return run(integral_constant<int, 2>{});
  if (T <= 32) return run(integral_constant<int, 4>{});
  return run(integral_constant<int, 8>{});
}
