// Decoding with several hypotheses (beams) per utterance: which continuations go on, and the caches that follow them.
//
//   beam_select    score[b, k] + x[b, k, v] - log sum_v exp x[b, k, v] over the K beams and V tokens of an utterance: the n best, the
//                  lowest k * V + v of equals.  Bound: reading the logits once (B * K * V * 2 bytes) in a large batch; one utterance's half a
//                  megabyte is bound by the latency of what follows.
//   beam_reorder   cache[.., b * K + k, .., t] = cache[.., b * K + parent[b, k], .., t] for t < length, in place: bound by memory, the
//                  rows that change written once and those they come from read once.
//
// The selection of an utterance is one cluster of 8 or 16 blocks and one launch, with no scratch in global memory, no counters
// that outlive the launch and no order of arrival in the result.  A warp reads a segment of one beam's row, 2048 values at a time in
// registers: their maximum and sum of exponentials, and the best n of the segment as a sorted list, one entry a lane.  Values enter
// the list only past a threshold (the n-th largest of the lanes' maxima, the list's n-th entry), which a handful of 2048 pass.
// A list entry is one word: the value as an ordered 16-bit number above the complement of its place in the segment, so that
// equal values sort by their place.  The blocks of the cluster read each other's maxima, sums and list heads: every block then knows each beam's
// normalisation (in 64 bits: the order of beams is decided by differences of sums) and the n-th best head, and sends what is no
// worse than that, n * n entries at most, to the first block, which ranks it.
#include "tcgen05.cuh"

namespace asrq {
namespace {

constexpr int kSelWarps = 8, kSelThreads = 32 * kSelWarps;
constexpr int kSelLists = 16 * kSelWarps;  // at most: one per warp of the cluster
constexpr int kSelMax = 32;                // beams, and continuations asked for
constexpr int kSelVecs = 8;                // 16-byte vectors a lane holds at a time
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
  float top;       // NaN or +inf: the row is no distribution
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

// Candidates of an utterance: a larger key first, of equals the smaller place (beam * V + token)
struct Cand {
  unsigned long long key;  // 0: none
  uint32_t place;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.key > b.key || (a.key == b.key && a.place < b.place); }

enum RowState { kRowLive = 0, kRowOver = 1, kRowNone = 2 };

template <bool bf16>
__global__ void __launch_bounds__(kSelThreads) beam_select_kernel(const SelectParams p) {
  __shared__ ListMeta meta[kSelWarps];
  __shared__ ListMeta all_meta[kSelLists];
  __shared__ uint32_t lists[kSelWarps][32];
  __shared__ Cand heads[kSelLists];
  __shared__ double row_norm[kSelMax];
  __shared__ double row_score[kSelMax];
  __shared__ int row_state[kSelMax];
  __shared__ Cand bound;
  __shared__ unsigned kept;
  __shared__ unsigned long long kept_key[kSelMax * kSelMax];
  __shared__ uint32_t kept_place[kSelMax * kSelMax];
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr uint32_t kNone = bf16 ? 0xff80u : 0xfc00u;  // -inf
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank, blocks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  const int b = int(blockIdx.x / blocks), n = p.n, K = p.K, V = p.V;
  const int n_lists = int(blocks) * kSelWarps, per_row = n_lists / K;  // warps of a row
  const int nvec = (V + 7) / 8, seg_vecs = (nvec + per_row - 1) / per_row;
  const int id = int(rank) * kSelWarps + warp, row = id / per_row, seg = id - row * per_row;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const volatile float* scores = p.scores + size_t(b) * K;
  const volatile uint8_t* over = p.finished ? p.finished + size_t(b) * K : nullptr;
  if (threadIdx.x == 0) kept = 0;
  if (threadIdx.x < K) {
    const float s = scores[threadIdx.x];
    row_score[threadIdx.x] = double(s);
    row_state[threadIdx.x] = !isfinite(s) ? kRowNone : over && over[threadIdx.x] ? kRowOver : kRowLive;
  }
  __syncthreads();

  uint32_t list = 0;             // this lane's entry of the warp's list, descending over the lanes
  float top = -INFINITY;         // of the warp's values so far
  double sum = 0.0;              // of exp(x - top), this lane's
  bool bad = false;
  if (row < K && row_state[row] == kRowLive) {
    const uint16_t* r = p.logits + size_t(b) * p.sb + size_t(row) * p.sk;
    const int v0 = seg * seg_vecs, v1 = min(nvec, v0 + seg_vecs);
#pragma unroll 1
    for (int vb = v0; vb < v1; vb += 32 * kSelVecs) {
      uint32_t x[kSelVecs][4];
#pragma unroll
      for (int i = 0; i < kSelVecs; ++i) {
        const int v = vb + i * 32 + lane;
        const uint4 u = v < v1 ? eight_of(r, v * 8, V, kNone) : make_uint4(kNone * 0x10001u, kNone * 0x10001u, kNone * 0x10001u, kNone * 0x10001u);
        x[i][0] = u.x, x[i][1] = u.y, x[i][2] = u.z, x[i][3] = u.w;
      }
      uint32_t mx = x[0][0];
#pragma unroll
      for (int i = 0; i < 4 * kSelVecs; ++i) mx = max2<bf16>(mx, x[i / 4][i % 4]);
      const float lo = out16_to_float(uint16_t(mx & 0xffffu), bf16), hi = out16_to_float(uint16_t(mx >> 16), bf16);
      bad |= !(fmaxf(lo, hi) < INFINITY) || lo != lo || hi != hi;
      const uint32_t best = ordered16(lo >= hi ? mx & 0xffffu : mx >> 16);  // this lane's largest
      const uint32_t by_lane = sort_descending(best, lane);
      const uint32_t least = __shfl_sync(0xffffffffu, by_lane, n - 1);      // n values of the chunk are at least this
      const float chunk_top = out16_to_float(unordered16(__shfl_sync(0xffffffffu, by_lane, 0)), bf16);
      const float now = fmaxf(top, chunk_top), ref = now > -INFINITY ? now : 0.f;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4 * kSelVecs; ++i) {
        const uint32_t w = x[i / 4][i % 4];
        acc[i % 2] += exp2_fast((out16_to_float(uint16_t(w & 0xffffu), bf16) - ref) * kLog2e);
        acc[2 + i % 2] += exp2_fast((out16_to_float(uint16_t(w >> 16), bf16) - ref) * kLog2e);
      }
      sum = sum * double(top > -INFINITY ? exp2f((top - ref) * kLog2e) : 0.f) + double((acc[0] + acc[1]) + (acc[2] + acc[3]));
      top = now;
      // what may enter the list
      const uint32_t floor16 = max(least, __shfl_sync(0xffffffffu, list, n - 1) >> 16);
      const uint32_t least2 = uint32_t(unordered16(floor16)) * 0x10001u;
      uint32_t hits[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 4 * kSelVecs; ++i) {
        const uint32_t m = ge2<bf16>(x[i / 4][i % 4], least2);
        hits[i / 16] |= ((m & 1u) | ((m >> 15) & 2u)) << (2 * (i % 16));
      }
      for (;;) {
        const bool have = (hits[0] | hits[1]) != 0;
        if (!__any_sync(0xffffffffu, have)) break;
        uint32_t entry = 0;
        if (have) {
          const int half = hits[0] ? 0 : 1, bit = __ffs(hits[half]) - 1, at = half * 32 + bit;  // value `at` of the lane's 64
          hits[half] &= hits[half] - 1;
          const int place = ((vb - v0) + (at / 8) * 32 + lane) * 8 + at % 8, token = v0 * 8 + place;
          if (token < V && place < (v1 - v0) * 8) entry = (ordered16(ld_x1(r + token)) << 16) | uint32_t(kSegValues - 1 - place);
        }
        const uint32_t last = __shfl_sync(0xffffffffu, list, n - 1);
        if (entry <= last) entry = 0;
        if (__any_sync(0xffffffffu, entry != 0)) list = merge_descending(list, sort_descending(entry, lane), lane);
      }
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  bad = __any_sync(0xffffffffu, bad);
  lists[warp][lane] = lane < n ? list : 0;
  if (lane == 0) {
    meta[warp].sum = sum;
    meta[warp].top = bad ? INFINITY : top;
    meta[warp].head = list;
  }
  tc::cluster_sync();
  for (int i = threadIdx.x; i < n_lists; i += kSelThreads) {
    const uint32_t at = tc::mapa(tc::smem_u32(&meta[i % kSelWarps]), uint32_t(i / kSelWarps));
    const float4 m = tc::ld_dsmem_v4(at);
    *reinterpret_cast<float4*>(&all_meta[i]) = m;
  }
  __syncthreads();
  for (int k = warp; k < K; k += kSelWarps) {  // a beam's normalisation
    if (row_state[k] != kRowLive) {
      if (lane == 0) row_norm[k] = 0.0;
      continue;
    }
    float t = -INFINITY;
    for (int i = lane; i < per_row; i += 32) t = fmaxf(t, all_meta[k * per_row + i].top);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    double s = 0.0;
    if (isfinite(t))
      for (int i = lane; i < per_row; i += 32) {
        const ListMeta& m = all_meta[k * per_row + i];
        if (m.top > -INFINITY) s += m.sum * exp(double(m.top) - double(t));
      }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      row_norm[k] = double(t) + log(s);
      if (!isfinite(t)) row_state[k] = kRowNone;
    }
  }
  __syncthreads();
  // entry `at` of list `l`; `word`: what the list holds there
  auto candidate = [&](int l, int at, uint32_t word) {
    const int k = l / per_row, sg = l - k * per_row;
    Cand c = {0, 0};
    if (k >= K) return c;
    const int state = row_state[k];
    if (state == kRowLive) {
      if (!word) return c;
      const uint32_t token = uint32_t(sg) * uint32_t(seg_vecs) * 8u + (kSegValues - 1 - (word & 0xffffu));
      const float x = out16_to_float(unordered16(word >> 16), bf16);
      c.key = ordered64(x > -INFINITY ? row_score[k] + (double(x) - row_norm[k]) : -INFINITY);
      c.place = uint32_t(k) * uint32_t(V) + token;
      return c;
    }
    // an ended beam: the end token at its own score, then the lowest others; a beam without hypothesis: the lowest tokens
    if (sg != 0 || at >= min(n, V)) return c;
    int token = at;
    double s = -INFINITY;
    if (state == kRowOver) {
      if (at == 0) s = row_score[k];
      token = at == 0 ? p.eos : at - 1 < p.eos ? at - 1 : at;
    }
    c.key = ordered64(s);
    c.place = uint32_t(k) * uint32_t(V) + uint32_t(token);
    return c;
  };
  if (threadIdx.x == 0) bound = Cand{0, 0xffffffffu};
  for (int l = threadIdx.x; l < n_lists; l += kSelThreads) heads[l] = candidate(l, 0, all_meta[l].head);
  __syncthreads();
  for (int l = threadIdx.x; l < n_lists; l += kSelThreads) {
    const Cand c = heads[l];
    if (!c.key) continue;
    int ahead = 0;
    for (int i = 0; i < n_lists; ++i) ahead += before(heads[i], c);
    if (ahead == n - 1) bound = c;  // one at most: no two candidates share a place
  }
  __syncthreads();
  {
    const Cand c = lane < n ? candidate(id, lane, lists[warp][lane]) : Cand{0, 0};
    const bool keep = c.key && !before(bound, c);
    const unsigned who = __ballot_sync(0xffffffffu, keep);
    if (who) {
      unsigned first = 0;
      if (lane == 0) {
        const uint32_t at = tc::mapa(tc::smem_u32(&kept), 0);
        asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(first) : "r"(at), "r"(unsigned(__popc(who))) : "memory");
      }
      first = __shfl_sync(0xffffffffu, first, 0) + __popc(who & ((1u << lane) - 1u));
      if (keep && first < kSelMax * kSelMax) {
        const uint32_t kat = tc::mapa(tc::smem_u32(&kept_key[first]), 0), pat = tc::mapa(tc::smem_u32(&kept_place[first]), 0);
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(kat), "l"(c.key) : "memory");
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(pat), "r"(c.place) : "memory");
      }
    }
  }
  tc::cluster_sync();
  if (rank != 0) return;
  const int m = int(min(kept, unsigned(kSelMax * kSelMax)));
  for (int i = threadIdx.x; i < m; i += kSelThreads) {
    const Cand c = {kept_key[i], kept_place[i]};
    int ahead = 0;
    for (int j = 0; j < m; ++j) ahead += before(Cand{kept_key[j], kept_place[j]}, c);
    if (ahead >= n) continue;
    const size_t o = size_t(b) * n + ahead;
    const int k = int(c.place / uint32_t(V)), token = int(c.place - uint32_t(k) * uint32_t(V));
    p.out_scores[o] = float(unordered64(c.key));
    p.parents[o] = k;
    p.tokens[o] = token;
    if (over) p.out_finished[o] = over[k] || token == p.eos;
  }
}

// One block per (layer and kind, utterance, head): a thread takes a 16-byte vector of one position in all beams, reads what moves
// and writes it, so no thread reads what another writes.
template <int MAXK>
__global__ void __launch_bounds__(256)
beam_reorder_kernel(uint4* __restrict__ cache, const long long* parents, const long long* length_dev, long long length, int K, int heads,
                    long long row_vecs, long long head_vecs, int pos_vecs, long long max_len, int B) {
  __shared__ int from[MAXK];
  __shared__ int moves;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h = blockIdx.x % heads;
  const long long lb = blockIdx.x / heads;
  const int b = int(lb % B);
  if (threadIdx.x == 0) moves = 0;
  __syncthreads();
  if (threadIdx.x < MAXK) {
    const int k = threadIdx.x;
    long long f = k < K ? *(const volatile long long*)(parents + (long long)b * K + k) : k;
    if (f < 0 || f >= K) f = k;  // no such beam: stays as it is
    from[k] = int(f);
    if (f != k) moves = 1;
  }
  __syncthreads();
  if (!moves) return;
  const long long len = min(max(length_dev ? *(const volatile long long*)length_dev : length, 0ll), max_len);
  uint4* base = cache + (lb * K * heads + h) * head_vecs;
  const long long n = len * pos_vecs;
  for (long long i = threadIdx.x; i < n; i += 256) {
    uint4 v[MAXK];
#pragma unroll
    for (int k = 0; k < MAXK; ++k)
      if (from[k] != k) v[k] = base[from[k] * row_vecs + i];
#pragma unroll
    for (int k = 0; k < MAXK; ++k)
      if (from[k] != k) base[k * row_vecs + i] = v[k];
  }
}

}  // namespace

bool beam_select_fits(int64_t K, int64_t V) {
  const int64_t per_row = kSelLists / K;  // sixteen blocks
  return ((V + 7) / 8 + per_row - 1) / per_row * 8 <= kSegValues;
}

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
  // sixteen blocks an utterance while eight would leave half of the chip idle, or where a segment of eight would be too long
  const int64_t per_row8 = 8 * kSelWarps / K;
  const bool wide = B * 16 <= sm_count || ((V + 7) / 8 + per_row8 - 1) / per_row8 * 8 > kSegValues;
  auto kern = dtype == ASRQ_BF16 ? beam_select_kernel<true> : beam_select_kernel<false>;
  if (wide) ASRQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(B * (wide ? 16 : 8)));
  cfg.blockDim = dim3(kSelThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = wide ? 16 : 8;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 1 : 2;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  return ASRQ_OK;
}

int beam_reorder(void* cache, const long long* parents, const long long* length_dev, int64_t length, int64_t L, int64_t B, int64_t K, int64_t heads,
                 int64_t max_len, int64_t pos_bytes, cudaStream_t stream) {
  auto kern = K <= 8 ? beam_reorder_kernel<8> : K <= 16 ? beam_reorder_kernel<16> : beam_reorder_kernel<32>;
  const int pos_vecs = int(pos_bytes / 16);
  const long long head_vecs = max_len * pos_vecs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(L * B * heads));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 0 : 1;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<uint4*>(cache), parents, length_dev, (long long)length, int(K), int(heads),
                                   heads * head_vecs, head_vecs, pos_vecs, (long long)max_len, int(B)));
  return ASRQ_OK;
}

}  // namespace asrq
