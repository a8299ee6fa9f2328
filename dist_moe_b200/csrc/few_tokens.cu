// The whole routed-expert layer for up to 64 tokens, in two launches and without routing tables in memory.
//
//   h[e, t] = c[t, e] * SwiGLU(W13[e] x[t]),   c[t, e] = sum of the scores of token t's routes to expert e   (bf16)
//   out[t]  = sum_e W2[e] h[e, t]                                                                            (bf16)
// Products and sums are in 32 bits; h is rounded once, with the score in it, so that the second launch sums over experts in its
// accumulators and has no weighted sum behind it.
//
// HBM bound: the weights of every expert that is hit stream through once (6 D F bytes each), all else is small.  So the weights never
// wait: each warp copies its pieces of them into shared memory kDepth items ahead (cp.async, 16 bytes a lane, read back by the same
// lane: no barrier), and the second launch starts under the first (programmatic dependent launch) and has its first pieces of W2 on
// their way before h is there.
//
// A block works on strips of 32 weight rows (16 features of gate and up; 32 output columns), its eight warps side by side on 32
// values of the inner dimension each.  An item is one such step of 256 values, 16 KiB; the items of all strips are dealt out evenly
// over the blocks, whatever the number of experts hit.  A strip that is cut between blocks is summed by the one of them that
// finishes last, in the order of the blocks.
//
// With so few columns the products are mma.sync m16n8k16, weights as the 16-row operand, tokens as the 8 columns: both operands are
// then loaded 16 bytes a lane along the inner dimension as they lie in memory, its order inside a step of 32 being the same for both
// (lane t of a row holds values 8 t .. 8 t + 7, in two instructions), and a gate value meets its up value in the same lane.
#include <type_traits>

#include "common.cuh"
#include "few_split.cuh"
#include "../../include/dist_moe_b200.h"

namespace dm {

constexpr int kFewTokens = DM_FEW_TOKENS_MAX;
constexpr int kFewExperts = 1024;
constexpr int kFewTopK = 32;
constexpr int kFewWarps = 8, kFewThreads = 32 * kFewWarps;
constexpr int kFewStep = 32 * kFewWarps;  // values of the inner dimension per item
constexpr int kFewRows = 32;              // weight rows per strip
constexpr int kFewItemBytes = 4 * kFewThreads * 16;

struct FewParams {
  const __nv_bfloat16* x;
  const void* ids;
  const void* scores;
  int ids_are_int64, scores_are_bf16;
  const __nv_bfloat16* w;  // W13 [E, 2F, D] or W2 [E, D, F]
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
  uint64_t* tokens;   // [E] bit t: token t
  int16_t* expert;    // [active]
  int16_t* base;      // [active + 1] first pair
  uint8_t* token;     // [pairs]
};
__host__ __device__ inline int few_active_bound(int T, int E, int K) { return T * K < E ? T * K : E; }
__host__ __device__ inline int few_table_bytes(int T, int E, int K) {
  const int active = few_active_bound(T, E, K);
  return (8 * E + 2 * active + 2 * (active + 1) + T * K + 15) / 16 * 16;
}

__device__ __forceinline__ int few_id(const FewParams& p, int i) {
  if (p.ids_are_int64) {
    const int64_t v = static_cast<const int64_t*>(p.ids)[i];
    return v >= 0 && v < p.E ? static_cast<int>(v) : v == -1 ? -1 : -2;
  }
  const int v = static_cast<const int32_t*>(p.ids)[i];
  return v >= 0 && v < p.E ? v : v == -1 ? -1 : -2;
}

__device__ __forceinline__ int few_tables(const FewParams& p, const FewTables& s, int* s_active, bool report) {
  for (int e = threadIdx.x; e < p.E; e += kFewThreads) s.tokens[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.K; i += kFewThreads) {
    const int id = few_id(p, i);
    if (id >= 0)
      atomicOr(reinterpret_cast<unsigned long long*>(&s.tokens[id]), 1ull << (i / p.K));
    else if (id == -2 && report)
      set_status(p.status, kInvalidExpertId, i);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int active = 0, pairs = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const uint64_t tokens = e0 + lane < p.E ? s.tokens[e0 + lane] : 0;
      const uint32_t hit = __ballot_sync(0xffffffffu, tokens != 0);
      int before = __popcll(tokens);
      const int own = before;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += v;
      }
      const int total = __shfl_sync(0xffffffffu, before, 31);
      if (tokens != 0) {
        const int at = active + __popc(hit & ((1u << lane) - 1));
        s.expert[at] = static_cast<int16_t>(e0 + lane);
        s.base[at] = static_cast<int16_t>(pairs + before - own);
        int n = pairs + before - own;
        for (uint64_t left = tokens; left != 0; left &= left - 1) s.token[n++] = static_cast<uint8_t>(__ffsll(static_cast<long long>(left)) - 1);
      }
      active += __popc(hit);
      pairs += total;
    }
    if (lane == 0) {
      s.base[active] = static_cast<int16_t>(pairs);
      *s_active = active;
    }
  }
  __syncthreads();
  return *s_active;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

template <bool kDown, int kTiles, int kDepth>
__global__ void __launch_bounds__(kFewThreads, kTiles > 4 ? 1 : 2) few_tokens_kernel(const FewParams p) {
  extern __shared__ __align__(128) uint8_t few_smem[];
  __shared__ int s_active, s_last;
  uint8_t* ring = few_smem;
  float* red = reinterpret_cast<float*>(few_smem + kDepth * kFewItemBytes);  // [warps][32 rows][8 * tiles]
  FewTables tab;
  tab.tokens = reinterpret_cast<uint64_t*>(few_smem + kDepth * kFewItemBytes + kFewWarps * kFewRows * 8 * kTiles * 4);
  tab.expert = reinterpret_cast<int16_t*>(tab.tokens + p.E);
  tab.base = tab.expert + few_active_bound(p.T, p.E, p.K);
  tab.token = reinterpret_cast<uint8_t*>(tab.base + few_active_bound(p.T, p.E, p.K) + 1);
  if (!kDown) dependents_may_start();
  const int active = few_tables(p, tab, &s_active, !kDown && blockIdx.x == 0);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
  const int inner = kDown ? p.F : p.D;
  const int steps = (inner + kFewStep - 1) / kFewStep;
  const int strips = kDown ? p.D / kFewRows : (p.F + 15) / 16;  // W13: of one expert
  const int length = kDown ? active * steps : steps;            // items of a strip
  const FewSplit split(kDown ? strips : static_cast<int64_t>(active) * strips, length, gridDim.x);
  const int64_t first = split.begin(blockIdx.x), end = split.end(blockIdx.x);
  const uint32_t own = smem_u32(ring) + threadIdx.x * 16;

  auto issue = [&](const FewCursor<kDown>& at, int slot) {
    const int k = at.c * kFewStep + warp * 32 + quad * 8;
    const bool in = k < inner;
    const int e = tab.expert[at.a];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int64_t r0, r1;
      if (kDown) {
        r0 = static_cast<int64_t>(e) * p.D + at.strip * kFewRows + 16 * i + g;
        r1 = r0 + 8;
      } else {
        const int f = min(at.strip * 16 + 8 * i + g, p.F - 1);  // beyond the last feature: computed, not kept
        r0 = static_cast<int64_t>(e) * 2 * p.F + f;
        r1 = r0 + p.F;
      }
      const int kk = in ? k : 0;
      cp_async16(own + (slot * 4 + 2 * i) * (kFewThreads * 16), p.w + r0 * inner + kk, in);
      cp_async16(own + (slot * 4 + 2 * i + 1) * (kFewThreads * 16), p.w + r1 * inner + kk, in);
    }
  };

  FewCursor<kDown> ahead, at;
  ahead.set(0, 1, 1, 1);
  if (first < end) ahead.set(first, strips, active, steps);
  at = ahead;
#pragma unroll
  for (int s = 0; s < kDepth; ++s) {
    if (first + s < end) {
      issue(ahead, s);
      ahead.next(strips, active, steps);
    }
    cp_async_commit();
  }
  if (kDown) {
    wait_for_launch_before();  // h is there from here on
    if (active == 0) {
      const int64_t n = static_cast<int64_t>(p.T) * p.D;
      for (int64_t i = blockIdx.x * static_cast<int64_t>(kFewThreads) + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kFewThreads)
        p.out[i] = __float2bfloat16_rn(0.f);
      return;
    }
  }
  if (first >= end) return;

  float acc[2][kTiles][4];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.f;
  };
  // The columns' rows of x or h for one expert, -1: none.
  int row[kTiles];
  int tiles = 0;
  auto columns = [&](int a) {
    const int base = tab.base[a], count = tab.base[a + 1] - base;
    if (kDown) {
      const uint64_t tokens = tab.tokens[tab.expert[a]];
      tiles = (p.T + 7) >> 3;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int t = 8 * n + g;
        row[n] = (tokens >> t) & 1 ? base + __popcll(tokens & ((1ull << t) - 1)) : -1;
      }
    } else {
      tiles = (count + 7) >> 3;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) row[n] = 8 * n + g < count ? tab.token[base + 8 * n + g] : -1;
    }
  };
  const __nv_bfloat16* source = kDown ? p.h : p.x;
  clear();
  columns(at.a);

  int slot = 0;
  int began = at.c + (kDown ? at.a * steps : 0);  // first item of the strip that this block has
  for (int64_t item = first; item < end; ++item) {
    const int k = at.c * kFewStep + warp * 32 + quad * 8;
    uint4 b[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      b[n] = make_uint4(0, 0, 0, 0);
      if (row[n] >= 0 && k < inner) b[n] = *reinterpret_cast<const uint4*>(source + static_cast<int64_t>(row[n]) * inner + k);
    }
    cp_async_wait<kDepth - 1>();
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = lds16(own + (slot * 4 + i) * (kFewThreads * 16));
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      if (n >= tiles) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_16x8x16(acc[i][n], w[2 * i].x, w[2 * i + 1].x, w[2 * i].y, w[2 * i + 1].y, b[n].x, b[n].y);
        mma_16x8x16(acc[i][n], w[2 * i].z, w[2 * i + 1].z, w[2 * i].w, w[2 * i + 1].w, b[n].z, b[n].w);
      }
    }
    if (item + kDepth < end) {
      issue(ahead, slot);
      ahead.next(strips, active, steps);
    }
    cp_async_commit();
    slot = slot + 1 == kDepth ? 0 : slot + 1;

    const FewCursor<kDown> done = at;
    at.next(strips, active, steps);
    const bool strip_end = kDown ? at.strip != done.strip : at.c == 0;
    if (strip_end || item + 1 == end) {
      // ---- sum over the warps -----------------------------------------------------------------------------------
      const int width = 8 * tiles;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        if (n >= tiles) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* to = red + (warp * kFewRows + 16 * i + g) * width + 8 * n + 2 * quad;
          *reinterpret_cast<float2*>(to) = make_float2(acc[i][n][0], acc[i][n][1]);
          *reinterpret_cast<float2*>(to + 8 * width) = make_float2(acc[i][n][2], acc[i][n][3]);
        }
      }
      __syncthreads();
      const int base = tab.base[done.a], count = kDown ? p.T : tab.base[done.a + 1] - base;
      const bool whole = strip_end && began == 0;
      const int64_t q = kDown ? done.strip : static_cast<int64_t>(done.a) * strips + done.strip;  // strip of the launch
      auto place = [&](int block) { return p.partial + split.place(block, q) * (kFewRows * 8 * kTiles); };
      auto sum_of = [&](int r, int col) {
        float v = 0.f;
#pragma unroll
        for (int w8 = 0; w8 < kFewWarps; ++w8) v += red[(w8 * kFewRows + r) * width + col];
        return v;
      };
      auto finish = [&](auto&& value) {
        if (kDown) {
          for (int i = threadIdx.x; i < kFewRows * count; i += kFewThreads) {
            const int r = i & (kFewRows - 1), col = i / kFewRows;
            p.out[static_cast<int64_t>(col) * p.D + done.strip * kFewRows + r] = __float2bfloat16_rn(value(r, col));
          }
        } else {
          for (int i = threadIdx.x; i < 16 * count; i += kFewThreads) {
            const int f = done.strip * 16 + (i & 15), col = i >> 4, r = 16 * ((i & 15) >> 3) + (i & 7);
            if (f >= p.F) continue;
            const int t = tab.token[base + col], e = tab.expert[done.a];
            float share = 0.f;
            for (int k1 = 0; k1 < p.K; ++k1)
              if (few_id(p, t * p.K + k1) == e)
                share += p.scores_are_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.scores)[t * p.K + k1])
                                           : static_cast<const float*>(p.scores)[t * p.K + k1];
            const float gate[1] = {value(r, col)}, up[1] = {value(r + 8, col)};
            float z[1];
            swiglu_f32(gate, up, z, p.act);
            p.h[static_cast<int64_t>(base + col) * p.F + f] = __float2bfloat16_rn(share * z[0]);
          }
        }
      };
      if (whole) {
        finish(sum_of);
      } else {
        float* mine = place(blockIdx.x);
        for (int i = threadIdx.x; i < kFewRows * width; i += kFewThreads) __stcg(mine + i, sum_of(i / width, i % width));
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          const int before = atomicAdd(p.arrived + q, 1);
          s_last = before == split.last_block(q) - split.first_block(q);
          if (s_last) p.arrived[q] = 0;  // clear for the next call
          __threadfence();
        }
        __syncthreads();
        if (s_last) {
          const int last = split.last_block(q);
          finish([&](int r, int col) {
            float v = 0.f;
            for (int block = split.first_block(q); block <= last; ++block) v += __ldcg(place(block) + r * width + col);
            return v;
          });
        }
      }
      __syncthreads();  // `red` may be written again
      clear();
      began = 0;
      if (item + 1 < end) columns(at.a);
    } else if (kDown && at.a != done.a) {
      columns(at.a);
    }
  }
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
  if (D % kFewRows != 0 || F % 8 != 0 || D > (1 << 20) || F > (1 << 20)) return kRcUnsupportedShape;
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
  auto run = [&](auto down_tag, auto tiles_tag, auto depth_tag) {
    constexpr bool down = decltype(down_tag)::value;
    constexpr int tiles = decltype(tiles_tag)::value, depth = decltype(depth_tag)::value;
    constexpr auto kernel = few_tokens_kernel<down, tiles, depth>;
    const size_t smem = depth * kFewItemBytes + kFewWarps * kFewRows * 8 * tiles * 4 + few_table_bytes(p.T, p.E, p.K);
    static PerDeviceOnce attr_set;
    const int arc = once_per_device(attr_set, [] {
      return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   depth * kFewItemBytes + kFewWarps * kFewRows * 8 * tiles * 4 +
                                                       few_table_bytes(kFewTokens, kFewExperts, kFewTopK)));
    });
    if (arc != 0) return arc;
    FewParams q = p;
    q.w = static_cast<const __nv_bfloat16*>(down ? w2 : w13);
    q.partial = reinterpret_cast<float*>(ws + (down ? l.partial2 : l.partial13));
    q.arrived = reinterpret_cast<int32_t*>(ws + (down ? l.arrived2 : l.arrived13));
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(kFewThreads);
    config.dynamicSmemBytes = smem;
    config.stream = static_cast<cudaStream_t>(stream);
    config.attrs = &attr;
    config.numAttrs = down ? 1 : 0;
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, q));
  };
  auto both = [&](auto tiles_tag, auto depth_tag) {
    const int first = run(std::false_type{}, tiles_tag, depth_tag);
    return first != 0 ? first : run(std::true_type{}, tiles_tag, depth_tag);
  };
  using std::integral_constant;
  if (T <= 8) return both(integral_constant<int, 1>{}, integral_constant<int, 6>{});
  if (T <= 16) return both(integral_constant<int, 2>{}, integral_constant<int, 5>{});
  if (T <= 32) return both(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  return both(integral_constant<int, 8>{}, integral_constant<int, 5>{});
}
