// The whole routed-expert layer for up to 64 tokens, in two launches and without routing tables in memory.
//
//   h[e, t] = c[t, e] * SwiGLU(W13[e] x[t]),   c[t, e] = sum of the scores of token t's routes to expert e   (bf16)
//   out[t]  = sum_e W2[e] h[e, t]                                                                            (bf16)
// Products and sums are in 32 bits; h is rounded once, with the score in it, so that the second launch sums over experts in its
// accumulators and has no weighted sum behind it.
//
// HBM bound: the weights of every expert that is hit stream through once (6 D F bytes each), all else is small.  So the weights never
// wait: one warp of a block brings them into a ring in shared memory (an item by one tensor copy), another the rows of x or h that meet
// them (512 bytes by one cp.async of the warp), and the second launch starts under the first (programmatic dependent launch) and has its first pieces of W2 on their way
// before h is there.
//
// A block works on strips of 32 weight rows (16 features of gate and up; 32 output columns); an item is 256 values of the inner
// dimension of a strip, 16 KiB.  The items of all strips are dealt out evenly over the blocks, whatever the number of experts hit.  A
// strip that is cut between blocks is summed by the one of them that finishes last, in the order of the blocks.  Of the eight warps
// that multiply, four share an item's inner dimension and two its rows.
//
// With so few columns the products are mma.sync m16n8k16, weights as the 16-row operand, tokens as the 8 columns: both operands are
// then read 16 bytes a lane along the inner dimension as they lie in shared memory, its order inside 32 values being the same for both
// (lane t of a row holds values 8 t .. 8 t + 7, in two instructions), and a gate value meets its up value in the same lane.  Row g of
// the instruction is row few_row(g) of the tile, which keeps the reads of the 128-byte swizzle free of bank conflicts.
#include <type_traits>

#include "few_split.cuh"
#include "gemm_common.cuh"
#include "../../include/dist_moe_b200.h"

namespace dm {

constexpr int kFewTokens = DM_FEW_TOKENS_MAX;
constexpr int kFewExperts = 1024;
constexpr int kFewTopK = 32;
constexpr int kFewWarps = 8, kFewKWarps = 4;       // that multiply; side by side along the inner dimension
constexpr int kFewThreads = 32 * (kFewWarps + 2);  // and one that loads weights, one that loads rows of x or h
constexpr int kFewStep = 64 * kFewKWarps;          // values of the inner dimension per item
constexpr int kFewRows = 32;                       // weight rows per strip
constexpr int kFewLineBytes = kFewRows * 128;      // weights of an item: four lines of 64 values, 32 rows each
constexpr int kFewWeightBytes = kFewKWarps * kFewLineBytes;
constexpr int kFewRowPitch = kFewStep * 2 + 64;    // rows of x or h: eight of them 16 bytes a lane hit every bank once
constexpr int kFewMaxDepth = 12;

struct FewParams {
  CUtensorMap tm_w;     // items: W13 (64 values, features, gate | up, lines, experts) or W2 (64 values, columns, lines, experts)
  CUtensorMap tm_tail;  // W2 with a last line of fewer than 64 values: (values, columns, experts)
  const __nv_bfloat16* x;
  const void* ids;
  const void* scores;
  int ids_are_int64, scores_are_bf16;
  __nv_bfloat16* h;        // [pairs of expert and token][F]
  float* partial;          // [blocks][2][kFewRows * 8 * tiles]
  int32_t* arrived;        // per strip, clear between calls
  __nv_bfloat16* out;
  int T, D, F, E, K;
  ActParams act;
  int* status;
};

// Which experts are hit, by which tokens: built by every block.
struct FewTables {
  uint64_t* tokens;  // [E] bit t: token t
  float* share;      // [pairs] c[t, e]; W13 only
  int16_t* expert;   // [active]
  int16_t* base;     // [active + 1] first pair
  int16_t* owner;    // [pairs] active expert
  int16_t* id;       // [T K]
  uint8_t* token;    // [pairs]
  __device__ __forceinline__ FewTables(uint8_t* at, int T, int E, int K) {
    const int active = T * K < E ? T * K : E;
    tokens = reinterpret_cast<uint64_t*>(at);
    share = reinterpret_cast<float*>(tokens + E);
    expert = reinterpret_cast<int16_t*>(share + T * K);
    base = expert + active;
    owner = base + active + 1;
    id = owner + T * K;
    token = reinterpret_cast<uint8_t*>(id + T * K);
  }
  static __host__ __device__ constexpr int bytes(int T, int E, int K) {
    return (8 * E + 9 * T * K + 4 * (T * K < E ? T * K : E) + 2 + 15) / 16 * 16;
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

// Returns the number of experts that are hit; `most` is the largest number of tokens of one.
__device__ __forceinline__ int few_tables(const FewParams& p, const FewTables& s, int (&s_found)[2], bool report, int& most) {
  for (int e = threadIdx.x; e < p.E; e += kFewThreads) s.tokens[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.K; i += kFewThreads) {
    const int id = few_id(p, i);
    s.id[i] = static_cast<int16_t>(id);
    if (id >= 0)
      atomicOr(reinterpret_cast<unsigned long long*>(&s.tokens[id]), 1ull << (i / p.K));
    else if (id == -2 && report)
      set_status(p.status, kInvalidExpertId, i);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int active = 0, pairs = 0, largest = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const uint64_t tokens = e0 + lane < p.E ? s.tokens[e0 + lane] : 0;
      const uint32_t hit = __ballot_sync(0xffffffffu, tokens != 0);
      const int own = __popcll(tokens);
      int before = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += v;
      }
      const int total = __shfl_sync(0xffffffffu, before, 31);
      if (tokens != 0) {
        const int at = active + __popc(hit & ((1u << lane) - 1));
        int n = pairs + before - own;
        s.expert[at] = static_cast<int16_t>(e0 + lane);
        s.base[at] = static_cast<int16_t>(n);
        for (uint64_t left = tokens; left != 0; left &= left - 1, ++n) {
          s.token[n] = static_cast<uint8_t>(__ffsll(static_cast<long long>(left)) - 1);
          s.owner[n] = static_cast<int16_t>(at);
        }
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
__device__ __forceinline__ void multipliers_meet() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kFewWarps) : "memory"); }
// Row g of the instruction: neighbouring ones differ in the swizzle's third bit.
__device__ __forceinline__ constexpr int few_row(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Where a block stands: strip, active expert, step of the inner dimension.  W13: strips of an expert follow one another; W2: the
// experts of a strip do, and are summed.
template <bool kDown>
struct FewCursor {
  int strip, a, c;
  __device__ __forceinline__ void set(int64_t item, int strips, int active, int steps) {
    c = static_cast<int>(item % steps);
    const int rest = static_cast<int>(item / steps);
    if (kDown) {
      a = rest % active;
      strip = rest / active;
    } else {
      strip = rest % strips;
      a = rest / strips;
    }
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

// kTiles: tiles of eight columns that the accumulators hold; kRed: those that meet in shared memory at a time.
template <bool kDown, int kTiles>
__global__ void __launch_bounds__(kFewThreads, kTiles > 1 ? 1 : 2) few_tokens_kernel(const __grid_constant__ FewParams p, int ring_bytes) {
  constexpr int kRed = kTiles > 2 ? 2 : kTiles;
  constexpr int kWidth = 8 * kRed;
  constexpr int kRedFloats = kFewKWarps * kFewRows * kWidth;
  extern __shared__ __align__(1024) uint8_t few_smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kFewMaxDepth], empty[kFewMaxDepth];
  __shared__ int s_found[2], s_last, abort_flag;
  float* red = reinterpret_cast<float*>(ring + ring_bytes);  // [2][warps along the inner dimension][32 rows][kWidth]
  const FewTables tab(ring + ring_bytes + 2 * kRedFloats * 4, p.T, p.E, p.K);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!kDown) dependents_may_start();
  if (warp == kFewWarps) {
    if (lane < kFewMaxDepth) {
      mbar_init(&full[lane], 1 + 32);  // the weights' warp and every lane of the rows' warp
      mbar_init(&empty[lane], kFewWarps);
    }
    if (lane == 0) {
      abort_flag = 0;
    }
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  int most;
  const int active = few_tables(p, tab, s_found, !kDown && blockIdx.x == 0, most);

  const int inner = kDown ? p.F : p.D;
  const int steps = (inner + kFewStep - 1) / kFewStep;
  const int strips = kDown ? p.D / kFewRows : (p.F + 15) / 16;  // W13: of one expert
  const int length = kDown ? active * steps : steps;            // items of a strip
  const FewSplit split(kDown ? strips : static_cast<int64_t>(active) * strips, length, gridDim.x);
  const int64_t first = split.begin(blockIdx.x);
  const int items = static_cast<int>(split.end(blockIdx.x) - first);
  // A place of the ring: 16 KiB of weights, and as many rows of x or h as the expert with the most tokens has.
  const int place_bytes = kFewWeightBytes + (most * kFewRowPitch + 1023) / 1024 * 1024;
  const int depth = min(kFewMaxDepth, ring_bytes / place_bytes);
  FewCursor<kDown> at;
  at.set(0, 1, 1, 1);
  if (items > 0) at.set(first, strips, active, steps);

  if (warp == kFewWarps) {
    // ======================= weights =======================
    const bool elected = elect_one();
    int place = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < items; ++i) {
      ok = warp_mbar_wait(&empty[place], phase ^ 1u, &abort_flag);
      if (!ok) break;
      uint8_t* to = ring + place * place_bytes;
      const int e = uniform(static_cast<int>(tab.expert[at.a])), strip = uniform(at.strip), c = uniform(at.c);
      const int lines = min(kFewKWarps, (inner - c * kFewStep + 63) / 64);
      if (elected) {
        if (kDown && (c + 1) * kFewStep > inner && (inner & 63) != 0) {
          mbar_arrive_expect_tx(&full[place], lines * kFewLineBytes);
          for (int l = 0; l < lines; ++l)
            tma_load_3d(to + l * kFewLineBytes, &p.tm_tail, c * kFewStep + 64 * l, strip * kFewRows, e, &full[place]);
        } else {
          mbar_arrive_expect_tx(&full[place], kFewWeightBytes);
          if (kDown)
            tma_load_4d(to, &p.tm_w, 0, strip * kFewRows, c * kFewKWarps, e, &full[place]);
          else
            tma_load_5d(to, &p.tm_w, 0, strip * 16, 0, c * kFewKWarps, e, &full[place]);
        }
      }
      __syncwarp();
      at.next(strips, active, steps);
      if (++place == depth) {
        place = 0;
        phase ^= 1u;
      }
    }
    if (lane == 0) {  // what is on its way has to land before the block gives its shared memory back
      if (!ok) set_status(p.status, kPipelineTimeout, 6, blockIdx.x);
      settle_ring(full, depth, ring_stop(place, phase), globaltimer_ns() + (ok ? 2000000000ull : kSettleNs));
    }
    return;
  }
  if (warp == kFewWarps + 1) {
    // ======================= rows of x or h =======================
    if (kDown) wait_for_launch_before();  // h is there from here on
    const uint32_t own = smem_u32(ring) + kFewWeightBytes + lane * 16;
    int place = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < items; ++i) {
      ok = warp_mbar_wait(&empty[place], phase ^ 1u, &abort_flag);
      if (!ok) break;
      const int k = at.c * kFewStep + lane * 8;
      const bool in = k < inner;
      const int base = tab.base[at.a], count = tab.base[at.a + 1] - base;
      const __nv_bfloat16* source = (kDown ? p.h + static_cast<int64_t>(base) * inner : p.x) + (in ? k : 0);
#pragma unroll 4
      for (int j = 0; j < count; ++j)
        cp_async16(own + place * place_bytes + j * kFewRowPitch, source + static_cast<int64_t>(kDown ? j : tab.token[base + j]) * inner, in);
      cp_async_arrive(&full[place]);
      at.next(strips, active, steps);
      if (++place == depth) {
        place = 0;
        phase ^= 1u;
      }
    }
    if (!ok && lane == 0) set_status(p.status, kPipelineTimeout, 8, blockIdx.x);
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ======================= products =======================
  if (kDown) {
    wait_for_launch_before();
    if (active == 0) {
      const int64_t n = static_cast<int64_t>(p.T) * p.D;
      for (int64_t i = blockIdx.x * static_cast<int64_t>(32 * kFewWarps) + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 32 * kFewWarps)
        p.out[i] = __float2bfloat16_rn(0.f);
      return;
    }
  } else {
    for (int i = threadIdx.x; i < tab.base[active]; i += 32 * kFewWarps) {
      const int t = tab.token[i], e = tab.expert[tab.owner[i]];
      float share = 0.f;
      for (int k = 0; k < p.K; ++k)
        if (tab.id[t * p.K + k] == e)
          share += p.scores_are_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.scores)[t * p.K + k])
                                     : static_cast<const float*>(p.scores)[t * p.K + k];
      tab.share[i] = share;
    }
  }
  const int g = lane >> 2, quad = lane & 3, kw = warp & (kFewKWarps - 1), half = warp / kFewKWarps;
  const int rho = few_row(g);
  // W13: rows 0 to 15 of a tile are gate features, 16 to 31 the same features of up
  const int r0 = kDown ? 16 * half + rho : 8 * half + rho, r1 = kDown ? r0 + 8 : r0 + 16;
  const uint32_t line = smem_u32(ring) + kw * kFewLineBytes;
  const uint32_t at_w = line + r0 * 128 + ((quad ^ rho) << 4);  // the other 32 values of the line: 64 bytes on or back
  const uint32_t at_b = smem_u32(ring) + kFewWeightBytes + kw * 128 + quad * 16;
  const int up = (r1 - r0) * 128;

  float acc[kTiles][4];
  auto clear = [&] {
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
  };
  // Columns: W13 the expert's tokens; W2 all tokens, those that are not the expert's being zero.
  int tiles = 0;
  int from[kTiles];  // offset of the column's row in a place; W2: -1 for none
  uint32_t hit = 0;  // W2: tiles that any token of the expert is in
  auto columns = [&](int a) {
    if (kDown) {
      const uint64_t tokens = tab.tokens[tab.expert[a]];
      tiles = (p.T + 7) >> 3;
      hit = 0;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int t = 8 * n + g;
        from[n] = (tokens >> t) & 1 ? __popcll(tokens & ((1ull << t) - 1)) * kFewRowPitch : -1;
        hit |= ((tokens >> (8 * n)) & 0xff) != 0 ? 1u << n : 0u;
      }
    } else {
      const int count = tab.base[a + 1] - tab.base[a];
      tiles = (count + 7) >> 3;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) from[n] = 8 * n + g < count ? (8 * n + g) * kFewRowPitch : -1;
      hit = (1u << tiles) - 1;
    }
  };
  clear();
  if (items > 0) columns(at.a);

  int place = 0, flip = 0;
  uint32_t phase = 0;
  int began = at.c + (kDown ? at.a * steps : 0);  // first item of the strip that this block has
  for (int item = 0; item < items; ++item) {
    // A wait that ran out is recorded; the block goes on without its data, so that its warps still meet.
    if (!warp_mbar_wait(&full[place], phase, &abort_flag) && lane == 0) set_status(p.status, kPipelineTimeout, 7, blockIdx.x);
    const uint32_t here = place * place_bytes;
    const int k = at.c * kFewStep + kw * 64;
    if (k < inner) {  // beyond the last value weights and rows are zero
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t aw = (at_w + here) ^ (h << 6);
        const uint4 lo = lds16(aw), hi = lds16(aw + up);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          if (((hit >> n) & 1) == 0) continue;
          uint4 b = make_uint4(0, 0, 0, 0);
          if (from[n] >= 0) b = lds16(at_b + here + h * 64 + from[n]);
          mma_16x8x16(acc[n], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
          mma_16x8x16(acc[n], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[place]);
    if (++place == depth) {
      place = 0;
      phase ^= 1u;
    }
    const FewCursor<kDown> done = at;
    at.next(strips, active, steps);
    const bool strip_end = kDown ? at.strip != done.strip : at.c == 0;
    if (!strip_end && item + 1 < items) {
      if (kDown && at.a != done.a) columns(at.a);
      continue;
    }
    // ---- sum over the warps, kRed tiles at a time, in two buffers in turn: one barrier each --------------------------
    const int base = tab.base[done.a], count = kDown ? p.T : tab.base[done.a + 1] - base;
    const bool whole = strip_end && began == 0;
    const int64_t q = kDown ? done.strip : static_cast<int64_t>(done.a) * strips + done.strip;  // strip of the launch
    auto part = [&](int block) { return p.partial + split.place(block, q) * (kFewRows * 8 * kTiles); };
    // `value(r, col)`: sum of weight row r of the strip and column col
    auto finish = [&](int col0, int cols, auto&& value) {
      if (kDown) {
        for (int i = threadIdx.x; i < kFewRows * cols; i += 32 * kFewWarps) {
          const int r = i & (kFewRows - 1), col = col0 + i / kFewRows;
          p.out[static_cast<int64_t>(col) * p.D + done.strip * kFewRows + r] = __float2bfloat16_rn(value(r, col));
        }
      } else {
        for (int i = threadIdx.x; i < 16 * cols; i += 32 * kFewWarps) {
          const int f = done.strip * 16 + (i & 15), col = col0 + (i >> 4);
          if (f >= p.F) continue;
          const float gate[1] = {value(i & 15, col)}, up1[1] = {value(16 + (i & 15), col)};
          float z[1];
          swiglu_f32(gate, up1, z, p.act);
          p.h[static_cast<int64_t>(base + col) * p.F + f] = __float2bfloat16_rn(tab.share[base + col] * z[0]);
        }
      }
    };
#pragma unroll
    for (int n0 = 0; n0 < kTiles; n0 += kRed) {
      if (n0 >= tiles) break;
      float* buf = red + flip * kRedFloats;
      flip ^= 1;
#pragma unroll
      for (int n = 0; n < kRed; ++n) {
        float* to = buf + (kw * kFewRows + r0) * kWidth + 8 * n + 2 * quad;
        *reinterpret_cast<float2*>(to) = make_float2(acc[n0 + n][0], acc[n0 + n][1]);
        *reinterpret_cast<float2*>(to + (r1 - r0) * kWidth) = make_float2(acc[n0 + n][2], acc[n0 + n][3]);
      }
      multipliers_meet();
      const int col0 = 8 * n0, cols = min(count - col0, kWidth);
      auto sum_of = [&](int r, int col) {
        float v = 0.f;
#pragma unroll
        for (int w4 = 0; w4 < kFewKWarps; ++w4) v += buf[(w4 * kFewRows + r) * kWidth + col - col0];
        return v;
      };
      if (whole) {
        finish(col0, cols, sum_of);
      } else {
        float* mine = part(blockIdx.x);
        for (int i = threadIdx.x; i < kFewRows * cols; i += 32 * kFewWarps) {
          const int r = i & (kFewRows - 1), col = col0 + i / kFewRows;
          __stcg(mine + col * kFewRows + r, sum_of(r, col));
        }
      }
    }
    if (!whole) {
      __threadfence();
      multipliers_meet();
      if (threadIdx.x == 0) {
        const int before = atomicAdd(p.arrived + q, 1);
        s_last = before == split.last_block(q) - split.first_block(q);
        if (s_last) p.arrived[q] = 0;  // clear for the next call
        __threadfence();
      }
      multipliers_meet();
      if (s_last) {
        const int begin = split.first_block(q), last = split.last_block(q);
        finish(0, count, [&](int r, int col) {
          float v = 0.f;
          for (int block = begin; block <= last; ++block) v += __ldcg(part(block) + col * kFewRows + r);
          return v;
        });
      }
    }
    clear();
    began = 0;
    if (item + 1 < items) columns(at.a);
  }
}

// An item of W13: (64 values, 16 features, gate and up, four lines); of W2: (64 values, 32 columns, four lines).  Beyond the last line or
// feature a box holds zeros.  `tail`: a line of W2 at a time, zeros beyond the last value.
static int few_encode(CUtensorMap* tm, const void* w, int64_t D, int64_t F, int64_t E, bool down, bool tail) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return kRcNoDriver;
  const cuuint64_t d = static_cast<cuuint64_t>(D), f = static_cast<cuuint64_t>(F), e = static_cast<cuuint64_t>(E);
  const cuuint64_t dims13[5] = {64, f, 2, d / 64, e}, strides13[4] = {2 * d, 2 * f * d, 128, 4 * f * d};
  const cuuint64_t dims2[4] = {64, d, f / 64, e}, strides2[3] = {2 * f, 128, 2 * f * d};
  const cuuint64_t dims_tail[3] = {f, d, e}, strides_tail[2] = {2 * f, 2 * f * d};
  const cuuint32_t box13[5] = {64, 16, 2, kFewKWarps, 1}, box2[4] = {64, kFewRows, kFewKWarps, 1}, box_tail[3] = {64, kFewRows, 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, tail ? 3 : down ? 4 : 5, const_cast<void*>(w),
                         tail ? dims_tail : down ? dims2 : dims13, tail ? strides_tail : down ? strides2 : strides13,
                         tail ? box_tail : down ? box2 : box13, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? kRcOk : 1000 + static_cast<int>(r);
}

struct FewLayout {
  int64_t arrived13, arrived2, partial13, partial2, h, total;
};
static FewLayout few_layout(int64_t T, int64_t D, int64_t F, int64_t E, int64_t K) {
  const int64_t active = T * K < E ? T * K : E;
  auto a128 = [](int64_t v) { return (v + 127) / 128 * 128; };
  const int64_t partial = a128(static_cast<int64_t>(sm_count()) * 2 * kFewRows * kFewTokens * 4);
  FewLayout l;
  l.arrived13 = 0;
  l.arrived2 = l.arrived13 + a128(active * ((F + 15) / 16) * 4);
  l.partial13 = l.arrived2 + a128(D / kFewRows * 4);
  l.partial2 = l.partial13 + partial;
  l.h = l.partial2 + partial;
  l.total = l.h + a128(T * K * F * 2);
  return l;
}
static int few_shape(int64_t T, int64_t D, int64_t F, int64_t E, int64_t K) {
  if (T <= 0 || D <= 0 || F <= 0 || E <= 0 || K <= 0) return kRcBadArg;
  if (T > kFewTokens || E > kFewExperts || K > kFewTopK) return kRcTooLarge;
  if (D % 64 != 0 || F % 8 != 0 || D > (1 << 20) || F > (1 << 20)) return kRcUnsupportedShape;
  return kRcOk;
}

}  // namespace dm

using namespace dm;

extern "C" int64_t dm_few_tokens_workspace_bytes(int64_t T, int64_t D, int64_t F, int E, int K) {
  const int rc = few_shape(T, D, F, E, K);
  return rc != kRcOk ? rc : few_layout(T, D, F, E, K).total;
}

extern "C" int dm_few_tokens(const void* x, const void* ids, int ids_are_int64, const void* scores, int scores_are_bf16,
                             const void* w13, const void* w2, void* out, int64_t T, int64_t D, int64_t F, int E, int K, int clamped,
                             float alpha, float limit, void* workspace, int64_t workspace_bytes, int num_sms, int* status,
                             void* stream) {
  if (!x || !ids || !scores || !w13 || !w2 || !out || !workspace) return kRcBadArg;
  int rc = few_shape(T, D, F, E, K);
  if (rc != kRcOk) return rc;
  for (const void* v : {x, w13, w2, static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(v) % 16 != 0) return kRcBadArg;
  const FewLayout l = few_layout(T, D, F, E, K);
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
  p.T = static_cast<int>(T), p.D = static_cast<int>(D), p.F = static_cast<int>(F), p.E = E, p.K = K;
  p.act = ActParams{clamped, alpha, limit};
  p.status = status;
  const unsigned grid = static_cast<unsigned>(persistent_grid(num_sms));
  auto run = [&](auto down_tag, auto tiles_tag) {
    constexpr bool down = decltype(down_tag)::value;
    constexpr int tiles = decltype(tiles_tag)::value;
    constexpr auto kernel = few_tokens_kernel<down, tiles>;
    constexpr int red = 2 * kFewKWarps * kFewRows * 8 * (tiles > 2 ? 2 : tiles) * 4;
    // Up to eight tokens a block leaves room for one of the other launch on its SM.
    constexpr int most = tiles > 1 ? 226 * 1024 : 112 * 1024;
    const int tables = FewTables::bytes(p.T, p.E, p.K);
    const int ring = (most - 1024 - red - tables) / 1024 * 1024;
    static PerDeviceOnce attr_set;
    const int arc = once_per_device(attr_set, [] {
      return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    });
    if (arc != 0) return arc;
    FewParams q = p;
    int erc = !down || F >= 64 ? few_encode(&q.tm_w, down ? w2 : w13, D, F, E, down, false) : kRcOk;
    if (erc == kRcOk && down && F % 64 != 0) erc = few_encode(&q.tm_tail, w2, D, F, E, true, true);
    if (erc != kRcOk) return erc;
    q.partial = reinterpret_cast<float*>(ws + (down ? l.partial2 : l.partial13));
    q.arrived = reinterpret_cast<int32_t*>(ws + (down ? l.arrived2 : l.arrived13));
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(kFewThreads);
    config.dynamicSmemBytes = 1024 + ring + red + tables;
    config.stream = static_cast<cudaStream_t>(stream);
    config.attrs = &attr;
    config.numAttrs = down ? 1 : 0;
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, q, ring));
  };
  auto both = [&](auto tiles_tag) {
    const int first = run(std::false_type{}, tiles_tag);
    return first != 0 ? first : run(std::true_type{}, tiles_tag);
  };
  using std::integral_constant;
  if (T <= 8) return both(integral_constant<int, 1>{});
  if (T <= 16) return both(integral_constant<int, 2>{});
  if (T <= 32) return both(integral_constant<int, 4>{});
  return both(integral_constant<int, 8>{});
}
