// Decoding with several hypotheses (beams) per utterance: which continuations go on, and the caches that follow them.
//
//   beam_select    score[b, k] + x[b, k, v] - log sum_v exp x[b, k, v] over the K beams and V tokens of an utterance: the n best, the
//                  lowest k * V + v of equals.  Bound: reading the logits once (B * K * V * 2 bytes) in a large batch; one utterance's half a
//                  megabyte is bound by the latency of what follows.
//   beam_reorder   cache[.., b * K + k, .., t] = cache[.., b * K + parent[b, k], .., t] for t < length, in place: bound by memory, the
//                  rows that change written once and those they come from read once.
//
// The selection of an utterance is one cluster of 2 to 16 blocks and one launch, with no scratch in global memory, no counters
// that outlive the launch and no order of arrival in the result.  A warp reads a segment of one beam's row, 1024 values at a time:
// each lane keeps the maximum and the sum of exponentials of its own values.  The warps of a block that share a row then agree on a value that
// n of the lanes' maxima reach, and only the lanes whose maximum does (n of the row's lanes in the block, if maxima differ) are read again, by
// the whole warp; what reaches it goes into the segment's list, of 32 entries at most, of which the best n are there.
// An entry is one word: the value as an ordered 16-bit number above the complement of its place in the segment, so that
// equal values sort by their place.  A row's segments do not depend on where it lies in memory, so beams with equal logits have equal
// sums.  The exponentials and the sums of 32 of them are in 32 bits, the exponential unit's, which is what bounds a large batch: it leaves a normalisation
// within 4e-6.  Maxima, sums and lists go to the first block of the cluster, which joins the sums in 64 bits (the order of beams is decided by their
// differences) and ranks what is no worse than a bound that n of the lists' best reach.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cluster_choice.h"
#include "tcgen05.cuh"

namespace asrq {

int ensure_dynamic_smem(const void* kernel, size_t bytes);

namespace {

constexpr int kSelWarps = 16, kSelThreads = 32 * kSelWarps;
constexpr int kSelLists = 16 * kSelWarps;  // at most: one per warp of the cluster
constexpr int kSelMax = 32;                // beams, and continuations asked for
constexpr int kSelVecs = 4;                // 16-byte vectors a lane holds at a time
constexpr int kSelWords = 4 * kSelVecs;
constexpr int kSelKept = 32 * kSelMax;     // candidates that are ranked: n lists of 32
constexpr int kSegValues = 65536;          // places that a list entry tells apart (beam_select_fits)

struct SelectParams {
  const uint16_t* logits;
  long long sb, sk;           // values between utterances and between beams
  const float* scores;        // B x K
  const uint8_t* finished;    // B x K, or NULL
  float* out_scores;          // B x n, as the rest
  long long *parents, *tokens;
  uint8_t* out_finished;
  int K, V, n, eos;
};

struct __align__(16) ListMeta {  // what a warp knows of its segment
  double sum;      // of exp(x - top)
  float top;       // +inf: the row is no distribution
  uint32_t head;   // its best entry, 0: none
};

template <bool bf16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // of both halves, a NaN wins
  if (bf16) {
    __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  return h2_as_u32(__hmax2_nan(u32_as_h2(a), u32_as_h2(b)));
}
template <bool bf16>
__device__ __forceinline__ uint32_t ge2(uint32_t a, uint32_t b) {  // 0xffff in each half where a >= b
  if (bf16) return __hge2_mask(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return __hge2_mask(u32_as_h2(a), u32_as_h2(b));
}
__device__ __forceinline__ float exp2_fast(float x) {  // two units in the last place
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t ordered16(uint32_t bits) {  // larger for the larger number; both zeros alike
  if (bits == 0x8000u) bits = 0;
  return bits & 0x8000u ? 0xffffu ^ bits : bits | 0x8000u;
}
__device__ __forceinline__ uint16_t unordered16(uint32_t o) { return uint16_t(o & 0x8000u ? o ^ 0x8000u : 0xffffu ^ o); }
__device__ __forceinline__ unsigned long long ordered64(double d) {
  if (d == 0.0) d = 0.0;
  const unsigned long long b = (unsigned long long)__double_as_longlong(d);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unordered64(unsigned long long o) {
  return __longlong_as_double((long long)(o >> 63 ? o ^ (1ull << 63) : ~o));
}

// A warp's 32 words in descending order of the lanes
__device__ __forceinline__ uint32_t exchange(uint32_t v, int lane, int stride, bool descending) {
  const uint32_t o = __shfl_xor_sync(0xffffffffu, v, stride);
  const bool low = (lane & stride) == 0;
  return low == descending ? max(v, o) : min(v, o);
}
__device__ __forceinline__ uint32_t sort_descending(uint32_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int stride = size / 2; stride >= 1; stride /= 2) v = exchange(v, lane, stride, (lane & size) == 0 || size == 32);
  return v;
}
__device__ __forceinline__ uint32_t merge_descending(uint32_t list, uint32_t sorted, int lane) {  // the best 32 of both
  uint32_t v = max(list, __shfl_sync(0xffffffffu, sorted, 31 - lane));
#pragma unroll
  for (int stride = 16; stride >= 1; stride /= 2) v = exchange(v, lane, stride, true);
  return v;
}

// Eight values of a row from value e on, -inf (`none`) past the row's end.  The row may start at any value: two aligned vectors
// that both lie inside the row, shifted together, or value by value at its ends.
__device__ __forceinline__ uint4 eight_of(const uint16_t* row, int e, int V, uint32_t none) {
  const uint16_t* at = row + e;
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(at)) & 15u;  // the same for all of a row's vectors
  if (off == 0 && e + 8 <= V) return ld_x4(at);
  const uint16_t* lo = at - off / 2;
  if (lo >= row && lo + 16 <= row + V) {
    const uint4 a = ld_x4(lo), b = ld_x4(lo + 8);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (off & 8u) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4u) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (off & 2u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = e + 2 * i < V ? ld_x1(at + 2 * i) : none, b = e + 2 * i + 1 < V ? ld_x1(at + 2 * i + 1) : none;
    w[i] = a | (b << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Vectors a and b of a row, eight values each, -inf past the row's end and in vectors from v1 on; the whole warp calls it.  The row may start at
// any value: a vector is two aligned ones, shifted together.  Those that lie inside the row are all on their way before the first is looked
// at, the two that its ends cut come value by value, a lane each.
struct TwoVectors {
  uint4 a, b;
};
template <bool bf16>
__device__ __forceinline__ TwoVectors vectors_of(const uint16_t* row, int va, int vb, int v1, int V) {
  constexpr uint32_t kNone = bf16 ? 0xff80u : 0xfc00u, kNone2 = kNone * 0x10001u;
  const int off = int(uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u) / 2, lane = threadIdx.x & 31;
  uint4 a[4];
  int first[4];
  bool wanted[4], cut = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int v = i < 2 ? va : vb;
    first[i] = (v + (i & 1)) * 8 - off;
    wanted[i] = v < v1 && (i % 2 == 0 || off != 0) && first[i] < V;
    a[i] = make_uint4(kNone2, kNone2, kNone2, kNone2);
    const bool in = first[i] >= 0 && first[i] + 8 <= V;
    if (wanted[i] && in) a[i] = ld_x4(row + first[i]);
    wanted[i] = wanted[i] && !in;
    cut |= wanted[i];
  }
  if (__any_sync(0xffffffffu, cut)) {
    const int last = (V - 1 + off) / 8, e = (lane < 8 ? 0 : last) * 8 + (lane & 7) - off;
    uint32_t x = lane < 16 && e >= 0 && e < V ? ld_x1(row + e) : kNone;
    x |= __shfl_down_sync(0xffffffffu, x, 1) << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = first[i] <= 0 ? 0 : 8;
      const uint4 end = make_uint4(__shfl_sync(0xffffffffu, x, from), __shfl_sync(0xffffffffu, x, from + 2), __shfl_sync(0xffffffffu, x, from + 4),
                                   __shfl_sync(0xffffffffu, x, from + 6));
      if (wanted[i]) a[i] = end;
    }
  }
  auto shifted = [&](const uint4& lo, const uint4& hi) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = off & 4 ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = off & 2 ? w[j + 1] : w[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], (off & 1) * 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  return {shifted(a[0], a[1]), shifted(a[2], a[3])};
}

// Candidates of an utterance: a larger key first, of equals the smaller place (beam * V + token)
struct __align__(16) Cand {
  unsigned long long key;  // 0: none
  uint32_t place, pad;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.key > b.key || (a.key == b.key && a.place < b.place); }
__device__ __forceinline__ Cand ld_cand(const Cand* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  return Cand{(unsigned long long)u.x | ((unsigned long long)u.y << 32), u.z, 0};
}

enum RowState { kRowLive = 0, kRowOver = 1, kRowNone = 2 };

constexpr float kLog2e = 1.4426950408889634f;
struct F2 {  // two 32-bit numbers that one instruction works on
  unsigned long long v;
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}

// The n largest of a warp's words, two a lane, all different (or 0: none), descending over the lanes
__device__ __forceinline__ uint32_t best_of(uint32_t a, uint32_t b, int n, int lane) {
  if (n > 12) return merge_descending(sort_descending(a, lane), sort_descending(b, lane), lane);
  uint32_t out = 0;
  for (int i = 0; i < n; ++i) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, max(a, b));
    if (a == m) a = 0;
    if (b == m) b = 0;
    if (lane == i) out = m;
  }
  return out;
}

// The n-th largest of a warp's 16-bit words; a sort for many (about the time of 12 maxima)
__device__ __forceinline__ uint32_t nth_of(uint32_t v, int n, int lane) {
  if (n > 12) return __shfl_sync(0xffffffffu, sort_descending(v, lane), n - 1);
  uint32_t key = v << 5 | uint32_t(lane), m = 0;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    m = __reduce_max_sync(0xffffffffu, key);
    if (key == m) key = 0;
  }
  return m >> 5;
}

struct SelectShared {  // of the first block, but for floors
  uint32_t floors[kSelWarps][8];     // each block: a warp's largest lane maxima
  uint8_t order[kSelWarps][32];      // each block: the lanes that a warp reads again
  ListMeta meta[kSelLists];
  uint32_t lists[kSelLists][kSelMax];
  Cand heads[kSelLists + kSelMax];   // of the lists, and of the beams that do not go on
  Cand kept[kSelKept];
  double row_norm[kSelMax], row_score[kSelMax];
  int row_state[kSelMax], live_row[kSelMax];
  uint8_t row_over[kSelMax];
  Cand bound;
  uint32_t edge;
  unsigned n_kept;
  int n_live;
};

template <bool bf16>
__global__ void __launch_bounds__(kSelThreads, 2) beam_select_kernel(const SelectParams p) {
  extern __shared__ __align__(16) uint8_t select_smem[];
  SelectShared& sh = *reinterpret_cast<SelectShared*>(select_smem);
  constexpr uint32_t kNone = bf16 ? 0xff80u : 0xfc00u;  // -inf
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank, blocks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  // the first block's shared memory is written by the others once it is known to run: arrived here, waited for before the first write
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int b = int(blockIdx.x / blocks), n = p.n, K = p.K, V = p.V;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const volatile float* scores = p.scores + size_t(b) * K;
  const volatile uint8_t* over = p.finished ? p.finished + size_t(b) * K : nullptr;
  const int nvec = (V + 7) / 8, n_lists = int(blocks) * kSelWarps, id = int(rank) * kSelWarps + warp;
  uint32_t y[kSelWords];  // the next values
  // (at_first: before the loop, where a row's ends may take registers; 1 utterance of 5 x 51866 values 9.1 -> 8.5 us)
  auto load = [&](const uint16_t* r, int vb, int v1, auto at_first) {
    const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(r)) & 15u;
    if (vb > 0 && vb + 32 * kSelVecs <= v1 && (vb + 32 * kSelVecs + 1) * 8 <= V) {  // all of it and its neighbours inside the row
      const uint16_t* lo = r + size_t(vb + lane) * 8 - off / 2;
      auto shifted = [&](auto words) {
#pragma unroll
        for (int i = 0; i < kSelVecs; ++i) {
          const uint4 a0 = ld_x4(lo + i * 256), a1 = ld_x4(lo + i * 256 + 8);
          const uint32_t w[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) y[4 * i + j] = __funnelshift_r(w[words.value + j], w[words.value + j + 1], (off & 2u) * 8u);
        }
      };
      if (off == 0) {
#pragma unroll
        for (int i = 0; i < kSelVecs; ++i) {
          const uint4 u = ld_x4(lo + i * 256);
          y[4 * i] = u.x, y[4 * i + 1] = u.y, y[4 * i + 2] = u.z, y[4 * i + 3] = u.w;
        }
      } else if (off < 4) {
        shifted(std::integral_constant<int, 0>{});
      } else if (off < 8) {
        shifted(std::integral_constant<int, 1>{});
      } else if (off < 12) {
        shifted(std::integral_constant<int, 2>{});
      } else {
        shifted(std::integral_constant<int, 3>{});
      }
      return;
    }
    if constexpr (decltype(at_first)::value) {
#pragma unroll
      for (int h = 0; h < kSelVecs; h += 2) {
        const TwoVectors u = vectors_of<bf16>(r, vb + h * 32 + lane, vb + h * 32 + 32 + lane, v1, V);
        y[4 * h] = u.a.x, y[4 * h + 1] = u.a.y, y[4 * h + 2] = u.a.z, y[4 * h + 3] = u.a.w;
        y[4 * h + 4] = u.b.x, y[4 * h + 5] = u.b.y, y[4 * h + 6] = u.b.z, y[4 * h + 7] = u.b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSelVecs; ++i) {
        const int v = vb + i * 32 + lane;
        const uint4 u = v < v1 ? eight_of(r, v * 8, V, kNone) : make_uint4(kNone * 0x10001u, kNone * 0x10001u, kNone * 0x10001u, kNone * 0x10001u);
        y[4 * i] = u.x, y[4 * i + 1] = u.y, y[4 * i + 2] = u.z, y[4 * i + 3] = u.w;
      }
    }
  };
  const float early = warp == 0 && lane < K ? scores[lane] : 0.f;
  const bool early_over = over && warp == 0 && lane < K && over[lane];
  // most often all beams go on: the first values as if they did, while the scores are on their way
  const int guess_per_row = n_lists / K, guess_row = id / guess_per_row;
  if (guess_row < K) {
    const int seg_vecs = (nvec + guess_per_row - 1) / guess_per_row, v0 = (id - guess_row * guess_per_row) * seg_vecs, v1 = min(nvec, v0 + seg_vecs);
    if (v0 < v1) load(p.logits + size_t(b) * p.sb + size_t(guess_row) * p.sk, v0, v1, std::true_type{});
  }
  if (warp == 0) {
    int state = kRowNone;
    if (lane < K) {
      state = !isfinite(early) ? kRowNone : early_over ? kRowOver : kRowLive;
      sh.row_score[lane] = double(early);
      sh.row_state[lane] = state;
      sh.row_over[lane] = early_over;
    }
    const unsigned live = __ballot_sync(0xffffffffu, state == kRowLive);
    if (state == kRowLive) sh.live_row[__popc(live & ((1u << lane) - 1u))] = lane;
    if (lane == 0) {
      sh.n_live = __popc(live);
      sh.n_kept = 0;
    }
  }
  __syncthreads();
  // the warps of the cluster share out the rows that go on
  const int n_live = sh.n_live, per_row = n_lists / max(n_live, 1), seg_vecs = (nvec + per_row - 1) / per_row;
  const int row_id = id / per_row, seg = id - row_id * per_row, v0 = seg * seg_vecs, v1 = min(nvec, v0 + seg_vecs);
  const bool works = row_id < n_live && v0 < v1;
  const uint16_t* r = works ? p.logits + size_t(b) * p.sb + size_t(sh.live_row[row_id]) * p.sk : nullptr;
  float top = -INFINITY;       // of the warp's values
  double sum = 0.0;            // of exp(x - top), this lane's
  uint32_t mine = kNone * 0x10001u;  // this lane's maximum, of low and high halves
  if (works) {
    if (!(row_id == guess_row && n_live == K)) load(r, v0, v1, std::false_type{});
#pragma unroll 1
    for (int vb = v0; vb < v1; vb += 32 * kSelVecs) {
      uint32_t x[kSelWords], mx = y[0];
#pragma unroll
      for (int i = 0; i < kSelWords; ++i) x[i] = y[i];
#pragma unroll
      for (int i = 1; i < kSelWords; ++i) mx = max2<bf16>(mx, x[i]);
      if (vb + 32 * kSelVecs < v1) load(r, vb + 32 * kSelVecs, v1, std::false_type{});
      mine = max2<bf16>(mine, mx);
      // (a NaN may pass as any maximum here: the row is no distribution then)
      const float lane_top = fmaxf(out16_to_float(uint16_t(mine & 0xffffu), bf16), out16_to_float(uint16_t(mine >> 16), bf16)), ref = lane_top > -INFINITY ? lane_top : 0.f;
      const F2 less(-ref, -ref), log2e(kLog2e, kLog2e);
      F2 acc[2] = {F2(0.f, 0.f), F2(0.f, 0.f)};
#pragma unroll
      for (int i = 0; i < kSelWords; ++i) {
        float d, e;
        ((F2(out16_to_float(uint16_t(x[i] & 0xffffu), bf16), out16_to_float(uint16_t(x[i] >> 16), bf16)) + less) * log2e).get(d, e);
        acc[i % 2] = acc[i % 2] + F2(exp2_fast(d), exp2_fast(e));
      }
      float s0, s1;
      (acc[0] + acc[1]).get(s0, s1);
      sum = sum * double(exp2_fast((top - ref) * kLog2e)) + double(s0 + s1);
      top = lane_top;
    }
  }
  const float lo = out16_to_float(uint16_t(mine & 0xffffu), bf16), hi = out16_to_float(uint16_t(mine >> 16), bf16);
  const bool bad = __any_sync(0xffffffffu, !(fmaxf(lo, hi) < INFINITY) || lo != lo || hi != hi);
  const uint32_t best = ordered16(lo >= hi ? mine & 0xffffu : mine >> 16);  // this lane's largest
  // the largest few of the lanes' for the block: of its warps on this row, 32 values at most
  const int w0 = max(warp - seg, 0), w1 = min(warp + per_row - seg, kSelWarps), each = min(8, 32 / (w1 - w0));
  const uint32_t most = __reduce_max_sync(0xffffffffu, best);
  {
    uint32_t key = best << 5 | uint32_t(lane);
#pragma unroll 1
    for (int i = 0; i < each; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, key);
      if (key == m) key = 0;
      if (lane == 0) sh.floors[warp][i] = m >> 5;
    }
  }
  {  // from the lanes' maxima to the warp's
    const float all = out16_to_float(unordered16(most), bf16);
    if (top > -INFINITY) sum *= double(exp2_fast((top - all) * kLog2e));
    top = bad ? INFINITY : all;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  __syncthreads();
  uint32_t list = 0;  // this lane's entry of the warp's list
  if (works && !bad) {
    uint32_t last = 0;  // n entries are no worse
    // n values of the row are at least `least`: of this warp's lanes, or of the first few of each of the block's warps on this row
    uint32_t least;
    if (each * (w1 - w0) >= n) {
      const uint32_t at = lane < each * (w1 - w0) ? *(const volatile uint32_t*)&sh.floors[w0 + lane / each][lane % each] : 0u;
      least = nth_of(at, n, lane);
    } else {
      least = nth_of(best, n, lane);
    }
    const uint32_t least2 = uint32_t(unordered16(least)) * 0x10001u;
    int waiting = 0;  // entries so far, at most 32, in no order
    volatile uint32_t* wait_at = sh.lists[warp];
    const unsigned again = __ballot_sync(0xffffffffu, best >= least);
    if (best >= least) sh.order[warp][__popc(again & ((1u << lane) - 1u))] = uint8_t(lane);
    __syncwarp();
    // every lane's values are `per` vectors; the warp takes 64 vectors of the chosen lanes at a time, the next ones on their way
    const int per = (v1 - v0 + 31) / 32, items = __popc(again) * per;
    int at_next[2];
    uint4 next[2];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int item = i0 + 32 * h + lane, v = item < items ? v0 + sh.order[warp][item / per] + 32 * (item % per) : v1;
        at_next[h] = v;
        next[h] = v < v1 ? eight_of(r, v * 8, V, kNone) : make_uint4(kNone * 0x10001u, kNone * 0x10001u, kNone * 0x10001u, kNone * 0x10001u);
      }
    };
    fetch(0);
#pragma unroll 1
    for (int i0 = 0; i0 < items; i0 += 64) {
      const uint4 u0 = next[0], u1 = next[1];
      const int v[2] = {at_next[0], at_next[1]};
      if (i0 + 64 < items) fetch(i0 + 64);
      const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
      uint32_t hits = 0;  // bit j: low half of word j, bit 16 + j: its high half
#pragma unroll
      for (int j = 0; j < 8; ++j) hits |= ge2<bf16>(w[j], least2) & (0x10001u << j);
      if (v[0] >= v1) hits &= 0xf0f0f0f0u;
      if (v[1] >= v1) hits &= 0x0f0f0f0fu;
      while (__any_sync(0xffffffffu, hits != 0)) {
        uint32_t entry = 0;
        if (hits) {
          const int bit = __ffs(hits) - 1, j = bit & 15, place = ((j < 4 ? v[0] : v[1]) - v0) * 8 + 2 * (j & 3) + (bit >> 4);
          hits &= hits - 1;
          uint32_t word = w[0];
#pragma unroll
          for (int x = 1; x < 8; ++x)
            if (j == x) word = w[x];
          if (v0 * 8 + place < V) entry = (ordered16(bit >> 4 ? word >> 16 : word & 0xffffu) << 16) | uint32_t(kSegValues - 1 - place);
        }
        if (entry <= last) entry = 0;
        const unsigned who = __ballot_sync(0xffffffffu, entry != 0);
        if (waiting + __popc(who) > 32) {  // only the best n stay
          __syncwarp();
          const uint32_t now = best_of(lane < waiting ? wait_at[lane] : 0u, entry, n, lane);
          __syncwarp();
          wait_at[lane] = now;
          waiting = n;
          last = __shfl_sync(0xffffffffu, now, n - 1);
          continue;
        }
        if (entry) wait_at[waiting + __popc(who & ((1u << lane) - 1u))] = entry;
        waiting += __popc(who);
      }
    }
    __syncwarp();
    list = lane < waiting ? wait_at[lane] : 0u;
  }
  const uint32_t head = __reduce_max_sync(0xffffffffu, list);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::mapa(tc::smem_u32(&sh.lists[id][lane]), 0)), "r"(list) : "memory");
  if (lane == 0)
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(tc::mapa(tc::smem_u32(&sh.meta[id]), 0)), "r"(uint32_t(__double2loint(sum))),
                 "r"(uint32_t(__double2hiint(sum))), "r"(__float_as_uint(top)), "r"(head)
                 : "memory");
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank != 0) return;
  for (int i = warp; i < n_live; i += kSelWarps) {  // a beam's normalisation
    const int k = sh.live_row[i];
    const ListMeta* of = sh.meta + i * per_row;
    float t = -INFINITY;
    for (int j = lane; j < per_row; j += 32) t = fmaxf(t, of[j].top);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    if (!isfinite(t)) {
      if (lane == 0) sh.row_state[k] = kRowNone;
      continue;
    }
    double s = 0.0;
    for (int j = lane; j < per_row; j += 32) s += of[j].sum * double(exp2_fast((of[j].top - t) * kLog2e));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sh.row_norm[k] = double(t) + log(s);
  }
  __syncthreads();
  auto of_list = [&](int l, uint32_t word) {  // an entry of list l
    const int i = l / per_row;
    Cand q = {0, 0, 0};
    if (i >= n_live || !word) return q;
    const int k = sh.live_row[i];
    if (sh.row_state[k] != kRowLive) return q;
    const uint32_t token = uint32_t(l - i * per_row) * uint32_t(seg_vecs) * 8u + (kSegValues - 1 - (word & 0xffffu));
    const float v = out16_to_float(unordered16(word >> 16), bf16);
    q.key = ordered64(v > -INFINITY ? sh.row_score[k] + (double(v) - sh.row_norm[k]) : -INFINITY);
    q.place = uint32_t(k) * uint32_t(V) + token;
    return q;
  };
  auto of_beam = [&](int k, int at) {  // an ended beam: the end token at its own score, then the lowest others; one without hypothesis: the lowest tokens
    Cand q = {0, 0, 0};
    if (k >= K || sh.row_state[k] == kRowLive || at >= min(n, V)) return q;
    int token = at;
    double s = -INFINITY;
    if (sh.row_state[k] == kRowOver) {
      if (at == 0) s = sh.row_score[k];
      token = at == 0 ? p.eos : at - 1 < p.eos ? at - 1 : at;
    }
    q.key = ordered64(s);
    q.place = uint32_t(k) * uint32_t(V) + uint32_t(token);
    return q;
  };
  // The heads, one a thread: of the lists, then of the beams that do not go on; neighbours to different warps.
  const int n_heads = n_lists + kSelMax, head_at = lane * kSelWarps + warp;
  const Cand head_cand = head_at < n_lists ? of_list(head_at, sh.meta[head_at].head) : of_beam(head_at - n_lists, 0);
  if (head_at < n_heads) sh.heads[head_at] = head_cand;
  __syncthreads();
  if (warp == 0) {  // the n-th largest of 32 lanes' maxima of heads: n candidates are no worse, by the high words alone
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kSelLists / 32 + 1; ++j)
      if (j * 32 < n_heads) most = max(most, uint32_t(sh.heads[j * 32 + lane].key >> 32));
    const uint32_t nth = __shfl_sync(0xffffffffu, sort_descending(most, lane), n - 1);
    if (lane == 0) sh.edge = nth;
  }
  __syncthreads();
  const uint32_t edge = sh.edge;
  Cand bound = {0, 0, 0};  // with a key: as well as the edge
  auto gather = [&]() {
    auto passes = [&](const Cand& q) { return q.key && uint32_t(q.key >> 32) >= edge && !(bound.key && before(bound, q)); };
    for (unsigned todo = __ballot_sync(0xffffffffu, head_at < n_heads && passes(head_cand)); todo; todo &= todo - 1) {
      const int l = (__ffs(todo) - 1) * kSelWarps + warp;
      const Cand q = l < n_lists ? of_list(l, sh.lists[l][lane]) : of_beam(l - n_lists, lane);
      const bool keep = passes(q);
      const unsigned who = __ballot_sync(0xffffffffu, keep);
      unsigned first = 0;
      if (lane == 0) first = atomicAdd(&sh.n_kept, unsigned(__popc(who)));
      first = __shfl_sync(0xffffffffu, first, 0) + __popc(who & ((1u << lane) - 1u));
      if (keep && first < kSelKept) sh.kept[first] = q;
    }
    __syncthreads();
  };
  gather();
  if (sh.n_kept > kSelKept) {
    // Equal high words beyond number: the n-th best head itself, which leaves n lists.
    if (head_at < n_heads && head_cand.key) {
      int ahead = 0;
      for (int j = 0; j < n_heads; ++j) ahead += before(ld_cand(&sh.heads[j]), head_cand);
      if (ahead == n - 1) sh.bound = head_cand;  // there is one: more than n heads pass, and no two share a place
    }
    __syncthreads();
    bound = ld_cand(&sh.bound);
    if (threadIdx.x == 0) sh.n_kept = 0;
    __syncthreads();
    gather();
  }
  // the n best, in order: eight lanes count what is ahead of a candidate
  const int m = int(min(sh.n_kept, unsigned(kSelKept))), part = lane & 7;
  for (int i0 = warp * 4; i0 < m; i0 += kSelThreads / 8) {
    const int i = i0 + lane / 8;
    const Cand q = i < m ? ld_cand(&sh.kept[i]) : Cand{0, 0, 0};
    int ahead = 0;
#pragma unroll 2
    for (int j = part; j < m; j += 8) ahead += before(ld_cand(&sh.kept[j]), q);
#pragma unroll
    for (int x = 1; x < 8; x *= 2) ahead += __shfl_xor_sync(0xffffffffu, ahead, x);
    if (i >= m || ahead >= n || part != 0) continue;
    const size_t o = size_t(b) * n + ahead;
    const int k = int(q.place / uint32_t(V)), token = int(q.place - uint32_t(k) * uint32_t(V));
    p.out_scores[o] = float(unordered64(q.key));
    p.parents[o] = k;
    p.tokens[o] = token;
    if (over) p.out_finished[o] = sh.row_over[k] || token == p.eos;
  }
}

// A run is what one (layer and kind, utterance, head) has to move in each of its beams: `length` positions, contiguous.  A warp a block, three an SM,
// each with its share of the runs in order; a chunk of a run is copied from every beam that another takes over into shared memory, and
// from there to every beam that takes one over, so each is read once, and all of it is read before any of it is written.  Copies and
// stores are bulk copies, four chunks under way.  (Loads and stores of threads ran at 4.5 to 5.8 TB/s of the row sizes tried, by block size
// and cache operator without a rule; this at 5.6 to 5.8 for runs of 100 and 224 positions in batches, 5.2 for one utterance's 59 MB in runs of 60; runs of a few positions are slower.)
constexpr int kMoveStages = 4, kMoveBytes = 16384, kMoveBlocks = 3;

struct ReorderParams {
  char* cache;
  const long long *parents, *length_dev;
  long long length, max_len, row_bytes, head_bytes, pos_bytes;
  int K, heads, B, L;
  unsigned* status;
};

__global__ void __launch_bounds__(32) beam_reorder_kernel(const ReorderParams p) {
  extern __shared__ __align__(128) uint8_t move_smem[];
  __shared__ __align__(8) unsigned long long full_bar[kMoveStages];
  const int lane = threadIdx.x;
  if (lane == 0) {
    for (int s = 0; s < kMoveStages; ++s) tc::mbar_init(tc::smem_u32(&full_bar[s]), 1);
    tc::fence_barrier_init();
  }
  __syncwarp();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long length = p.length_dev ? *(const volatile long long*)p.length_dev : p.length;
  const long long run = min(max(length, 0ll), p.max_len) * p.pos_bytes;
  const int runs_of = p.L * p.heads, items = runs_of * p.B;  // of an utterance; of all, utterance by utterance
  const int share = (items + int(gridDim.x) - 1) / int(gridDim.x), end = min(items, (int(blockIdx.x) + 1) * share);
  struct Cursor {
    int item, b;         // run; the utterance that what follows is of
    long long off;       // in the run
    int parent, chunk;   // this lane's beam's parent; bytes copied from a beam at a time
    unsigned moves, from;  // beams that take another over; beams that are taken over
  };
  auto find = [&](Cursor& c) {  // to the next run with something to move
    while (c.item < end && run > 0) {
      const int b = c.item / runs_of;
      if (b != c.b) {
        c.b = b;
        long long f = lane < p.K ? *(const volatile long long*)(p.parents + (long long)b * p.K + lane) : lane;
        if (f < 0 || f >= p.K) f = lane;  // no such beam: stays as it is
        c.parent = int(f);
        c.moves = __ballot_sync(0xffffffffu, c.parent != lane);
        c.from = __reduce_or_sync(0xffffffffu, c.parent != lane ? 1u << c.parent : 0u);
        c.chunk = (kMoveBytes / max(1, __popc(c.from))) & ~127;
      }
      if (c.moves) return true;
      c.item = min(end, (b + 1) * runs_of);
    }
    return false;
  };
  auto step = [&](Cursor& c) {
    c.off += c.chunk;
    if (c.off >= run) {
      c.off = 0;
      ++c.item;
    }
  };
  auto place = [&](const Cursor& c) {
    const int x = c.item - c.b * runs_of, l = x / p.heads;
    return p.cache + ((long long)l * p.B + c.b) * p.K * p.row_bytes + (x - l * p.heads) * p.head_bytes + c.off;
  };
  auto bytes_of = [&](const Cursor& c) { return uint32_t(min((long long)c.chunk, run - c.off)); };
  Cursor in = {int(blockIdx.x) * share, -1, 0, 0, 0, 0, 0}, out = in;
  int started = 0;
  auto start = [&]() {  // the next chunk's copies
    const int s = started % kMoveStages;
    const uint32_t bytes = bytes_of(in), bar = tc::smem_u32(&full_bar[s]), to = tc::smem_u32(move_smem) + uint32_t(s * kMoveBytes);
    if (lane == 0) {
      tc::mbar_arrive_expect_tx(bar, bytes * __popc(in.from));
      const char* at = place(in);
      int slot = 0;
      for (unsigned m = in.from; m; m &= m - 1, ++slot)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to + uint32_t(slot * in.chunk)),
                     "l"(at + (__ffs(m) - 1) * p.row_bytes), "r"(bytes), "r"(bar)
                     : "memory");
    }
    step(in);
    ++started;
  };
  for (int s = 0; s < kMoveStages - 1 && find(in); ++s) start();
  int done = 0;
  bool ok = true;
  for (; ok && find(out); ++done) {
    const int s = done % kMoveStages;
    ok = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&full_bar[s]), uint32_t(done / kMoveStages) & 1u, p.status, 81));
    if (!ok) break;
    const uint32_t bytes = bytes_of(out), from = tc::smem_u32(move_smem) + uint32_t(s * kMoveBytes);
    char* at = place(out);
    for (unsigned m = out.moves; m; m &= m - 1) {
      const int k = __ffs(m) - 1, f = __shfl_sync(0xffffffffu, out.parent, k), slot = __popc(out.from & ((1u << f) - 1u));
      if (lane == 0)
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(at + k * p.row_bytes), "r"(from + uint32_t(slot * out.chunk)), "r"(bytes)
                     : "memory");
    }
    if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    step(out);
    if (find(in)) {  // into the stage that the chunk before this one has left
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      __syncwarp();
      start();
    }
  }
  for (; done < started && !ok; ++done)  // copies that are on their way still land here
    tc::mbar_wait(tc::smem_u32(&full_bar[done % kMoveStages]), uint32_t(done / kMoveStages) & 1u, p.status, 82);
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

}  // namespace

// whether the segments of a cluster of `blocks` are short enough for their lists
bool segments_fit(int64_t blocks, int64_t K, int64_t V) {
  const int64_t per_row = blocks * kSelWarps / K;
  return per_row > 0 && ((V + 7) / 8 + per_row - 1) / per_row * 8 <= kSegValues;
}
// Whether the current device holds clusters of 16 blocks of the selection: asked once for each device and kernel, which the answer also allows them
int holds_clusters_of_16(void (*kern)(SelectParams), bool bf16, bool* holds) {
  static std::atomic<uint64_t> asked[2], held[2];  // by device
  int dev = 0;
  ASRQ_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(asked[bf16].load(std::memory_order_acquire) & bit)) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = sizeof(SelectShared);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    if (n > 0) held[bf16].fetch_or(bit, std::memory_order_relaxed);
    asked[bf16].fetch_or(bit, std::memory_order_release);
  }
  *holds = (held[bf16].load(std::memory_order_relaxed) & bit) != 0;
  return ASRQ_OK;
}

bool beam_select_fits(int64_t K, int64_t V) { return segments_fit(8, K, V); }

int beam_select(const void* logits, int64_t sb, int64_t sk, const float* scores, const uint8_t* finished, int64_t eos, float* out_scores,
                long long* parents, long long* tokens, uint8_t* out_finished, int64_t B, int64_t K, int64_t V, int64_t n, int dtype, int sm_count,
                cudaStream_t stream) {
  SelectParams p = {};
  p.logits = static_cast<const uint16_t*>(logits);
  p.sb = sb;
  p.sk = sk;
  p.scores = scores;
  p.finished = finished;
  p.out_scores = out_scores;
  p.parents = parents;
  p.tokens = tokens;
  p.out_finished = out_finished;
  p.K = int(K);
  p.V = int(V);
  p.n = int(n);
  p.eos = int(eos);
  auto kern = dtype == ASRQ_BF16 ? beam_select_kernel<true> : beam_select_kernel<false>;
  int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), sizeof(SelectShared));
  if (rc) return rc;
  bool holds_16 = false;
  if ((rc = holds_clusters_of_16(kern, dtype == ASRQ_BF16, &holds_16))) return rc;
  const int blocks = choose_select(B, sm_count, holds_16, [&](int n) { return segments_fit(n, K, V); });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(B * blocks));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = sizeof(SelectShared);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(blocks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 1 : 2;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  return ASRQ_OK;
}

int beam_reorder(void* cache, const long long* parents, const long long* length_dev, int64_t length, int64_t L, int64_t B, int64_t K, int64_t heads,
                 int64_t max_len, int64_t pos_bytes, void* status, int sm_count, cudaStream_t stream) {
  ReorderParams p = {};
  p.cache = static_cast<char*>(cache);
  p.parents = parents;
  p.length_dev = length_dev;
  p.length = length;
  p.max_len = max_len;
  p.pos_bytes = pos_bytes;
  p.head_bytes = max_len * pos_bytes;
  p.row_bytes = heads * p.head_bytes;
  p.K = int(K), p.heads = int(heads), p.B = int(B), p.L = int(L);
  p.status = static_cast<unsigned*>(status);
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(beam_reorder_kernel), kMoveStages * kMoveBytes);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(std::min<int64_t>(int64_t(kMoveBlocks) * sm_count, L * B * heads)));
  cfg.blockDim = dim3(32);
  cfg.dynamicSmemBytes = kMoveStages * kMoveBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 0 : 1;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, beam_reorder_kernel, p));
  return ASRQ_OK;
}

}  // namespace asrq
