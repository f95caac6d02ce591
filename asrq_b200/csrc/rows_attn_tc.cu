// Attention of many query rows over keys that they share, on the 5th-generation tensor cores: the tokens of a prompt over an encoder's
// states, or the rows of many beams or samples over their prompt.
//
// A block holds 128 rows (all query heads of a key head, so several tokens or beams) and walks its keys 96 (64 with 128 dimensions) at a
// time: S = Q K^T into tensor memory, a thread per row reads its scores, and writes the weights 2^(scale' s - m + lift) in 16 bits to tensor memory
// too, from where O += P V takes them as its first operand.  K arrives by TMA as rows of the contraction, V as it lies, dimensions
// contiguous, which the second operand's descriptor calls MN-major.  The next S is on its way as soon as the scores are in registers, and
// two blocks an SM fill each other's waits.  Blocks stay and take one item after the other: the next one's queries and keys arrive and its first S is
// done while the last weights and the result of the one before are.
// The reference exponent m of a row moves only when its maximum has grown by more than 8 (bf16; 4 in fp16, see weight_growth): a sum in 32 bits has
// room for that, and O is scaled at the first tiles and hardly ever after.
// The weights are rounded to the values' type, which is what the second product takes (a second one of their remainders would double it): half a step
// each, against which the polynomial's 2.6e-6 does not count.
// A row's sum is that of the weights as they are rounded, or an average of equal values would not be that value: P times 16 columns of
// ones, into tensor memory like O (16 x 224 rows on 1500 keys: 56.0 us; 65.9 with threads adding up what they have rounded).
//
// Bound: at 64 dimensions the exponentials, 16 a cycle and SM, of which every fourth pair goes to the multipliers instead; at 128 these and the
// memory's bytes where few rows share many keys.
#include <algorithm>
#include <type_traits>

#include "rows_attn.cuh"

namespace asrq {

int ensure_dynamic_smem(const void* kernel, size_t bytes);

namespace {

struct FlashParams {
  uint16_t* out;
  const long long* len;
  float *parts, *stats;  // as in RowsParams
  unsigned* status;
  long long keys;
  int R, G, Hkv, tiles, units, whole, split, slots, part_rows, k_batch, v_batch, k_head, v_head;  // *_batch, *_head: 0 where all utterances or heads share them
  // units: what a block takes at a time; the first `whole` are items, the others parts of items, `split` of each; slots: parts of an item there is room for
  float scale_log2;  // positive
};

template <int HD>
struct FlashLayout {
  static constexpr int kKeys = HD == 64 ? 96 : 64;  // of a tile: tensor memory has 256 columns for S (32 bits), P (16 bits) and O of a block
  static constexpr int kStages = HD == 64 ? 3 : 2;
  static constexpr int kQ = kTcRows * HD * 2, kTile = kKeys * HD * 2;
  static constexpr int kOnesBytes = 2048;  // 16 rows of 128 bytes
  static constexpr int kK = kQ, kV = kQ + kStages * kTile, kOnes = kQ + 2 * kStages * kTile, kBars = kOnes + kOnesBytes;
  static constexpr int kBytes = kBars + (4 * kStages + 7) * 8 + 16 + 1024;  // 1024: the base is aligned to it
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, int c4, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}
// MN-major operand with 128-byte swizzle: 64 values along N contiguous, 8 k apart by 128 bytes each, groups of 8 k 1024 bytes apart; the
// next 64 values along N `block` bytes on.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t block) {
  uint64_t d = 0;
  d |= uint64_t((addr & 0x3ffffu) >> 4);
  d |= uint64_t((block & 0x3ffffu) >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// one column of tensor memory, 32 lanes of the warp's quadrant
__device__ __forceinline__ uint32_t tmem_ld_32x1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}
__device__ __forceinline__ void tmem_st_32x1(uint32_t taddr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory");
}
// registers to tensor memory: 32 lanes of the warp's quadrant x 16 columns
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
      "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ unsigned long long two(float a, float b) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}

// 2^x of a pair without the exponential unit, x at most 100 and below -126 as -126: x = i + f with a whole i and f within a half (adding 1.5 * 2^23
// leaves i in the low bits), 2^f by the polynomial of degree 4 with the least relative error there (Remez' exchange: 2.6e-6), times 2^i.
__device__ __forceinline__ unsigned long long ex2_poly(unsigned long long x) {
  constexpr float kShift = 12582912.f + 127.f;  // the exponent's bias with it
  constexpr float c0 = 0.9999992847442627f, c1 = 0.6931217908859253f, c2 = 0.240247443318367f, c3 = 0.05591785907745361f, c4 = 0.009570102207362652f;
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(lo));  // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(hi));
  x = two(lo, hi);
  unsigned long long i = x, f = x, y = two(c4, c4);
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(i) : "l"(two(kShift, kShift)));
  unsigned long long whole = i;
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(whole) : "l"(two(-kShift, -kShift)));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(f) : "l"(whole), "l"(two(-1.f, -1.f)));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(y) : "l"(f), "l"(two(c3, c3)));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(y) : "l"(f), "l"(two(c2, c2)));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(y) : "l"(f), "l"(two(c1, c1)));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(y) : "l"(f), "l"(two(c0, c0)));
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(i));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(two(__uint_as_float(a << 23), __uint_as_float(b << 23))));
  return y;
}

// Most waits find their phase over: a test first, which unlike try_wait never suspends the warp.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, unsigned* status, unsigned site) {
  return tc::mbar_test_wait(bar, parity) || tc::mbar_wait(bar, parity, status, site);
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(192, 2)
flash_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ FlashParams p) {
  using L = FlashLayout<HD>;
  constexpr int ST = L::kStages, HALVES = HD / 64, kKeys = L::kKeys;
  constexpr uint32_t kP = kKeys, kOut = 256 - HD, kSum = kOut - 16;  // columns of tensor memory: the scores from 0, the weights, their sum (16 times), the result
  static_assert(kP + kKeys / 2 <= kSum, "256 columns");
  extern __shared__ uint8_t flash_smem[];
  const uint32_t base = (tc::smem_u32(flash_smem) + 1023u) & ~1023u;
  uint8_t* smem = flash_smem + (base - tc::smem_u32(flash_smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [&](int i) { return base + L::kBars + uint32_t(i) * 8u; };
  auto k_full = [&](int s) { return bar(s); };
  auto k_free = [&](int s) { return bar(ST + s); };
  auto v_full = [&](int s) { return bar(2 * ST + s); };
  auto v_free = [&](int s) { return bar(3 * ST + s); };
  const uint32_t s_full = bar(4 * ST), s_free = bar(4 * ST + 1), p_full = bar(4 * ST + 2), o_done = bar(4 * ST + 3), q_full = bar(4 * ST + 4), o_free = bar(4 * ST + 5), q_free = bar(4 * ST + 6);
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + L::kBars + (4 * ST + 7) * 8);

  if (threadIdx.x < L::kOnesBytes / 16) {
    constexpr uint32_t one2 = BF16 ? 0x3f803f80u : 0x3c003c00u;
    tc::st_shared_v4(base + L::kOnes + threadIdx.x * 16u, one2, one2, one2, one2);
    tc::fence_proxy_async_smem();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4 * ST + 7; ++i) {
      const uint32_t x = bar(i);
      tc::mbar_init(x, x == s_free || x == p_full || x == o_free ? 4 : 1);  // from each softmax warp
    }
    tc::fence_barrier_init();
    tc::prefetch_tmap(&qmap);
    tc::prefetch_tmap(&kmap);
    tc::prefetch_tmap(&vmap);
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  struct Unit {
    int b, h, row0, rows, rest;     // rest: which part in memory, negative: the result itself
    int t0, n, last_keys;           // its tiles of keys, and the keys of the last one
  };
  auto unit = [&](int u) {
    Unit w;
    const bool alone = u < p.whole;
    const int rest = u - p.whole, split = alone ? 1 : p.split, at = alone ? 0 : rest / split, part = alone ? 0 : rest - at * split;
    const int item = alone ? u : p.whole + at, bh = item / p.tiles;
    w.rest = alone || !p.parts ? -1 : at * p.slots + part;
    w.b = bh / p.Hkv;
    w.h = bh - w.b * p.Hkv;
    w.row0 = (item - bh * p.tiles) * kTcRows;
    w.rows = min(kTcRows, p.R * p.G - w.row0);
    const long long n_keys = p.len ? min(max(*(const volatile long long*)(p.len + w.b), 0ll), p.keys) : p.keys;
    // (fewer than 2^25 tiles, at most 64 parts)
    const unsigned all = unsigned((n_keys + kKeys - 1) / kKeys);
    w.t0 = int(all * unsigned(part) / unsigned(split));
    w.n = int(all * unsigned(part + 1) / unsigned(split)) - w.t0;
    w.last_keys = w.t0 + w.n == int(all) ? int(n_keys - (long long)(int(all) - 1) * kKeys) : kKeys;
    return w;
  };
  const int step = int(gridDim.x);

  if (warp == 0) {  // the copies, tile by tile through all units
    if (lane == 0) {
      bool ok = true;
      int t = 0, v_started = 0, taken = 0;
      for (int x = int(blockIdx.x); x < p.units && ok; x += step) {
        const Unit w = unit(x);
        const int kb = p.k_batch ? w.b : 0, kh = p.k_head ? w.h : 0, vb = p.v_batch ? w.b : 0, vh = p.v_head ? w.h : 0;
        for (int j = 0; j < w.n; ++j, ++t) {
          const int s = t % ST, at = (w.t0 + j) * kKeys;
          const uint32_t ph = (uint32_t(t / ST) & 1u) ^ 1u;
          ok = wait(k_free(s), ph, p.status, 61);
          if (!ok) break;
          tc::mbar_arrive_expect_tx(k_full(s), L::kTile);
          for (int i = 0; i < HALVES; ++i) tma_load_4d(base + L::kK + uint32_t(s * L::kTile + i * kKeys * 128), &kmap, i * 64, at, kh, kb, k_full(s));
          ok = wait(v_free(s), ph, p.status, 62);
          if (!ok) {
            ++t;
            break;
          }
          tc::mbar_arrive_expect_tx(v_full(s), L::kTile);
          for (int i = 0; i < HALVES; ++i) tma_load_4d(base + L::kV + uint32_t(s * L::kTile + i * kKeys * 128), &vmap, i * 64, at, vh, vb, v_full(s));
          ++v_started;
          if (j == 0) {  // the queries' place: free when the last scores of the unit before are done
            if (taken > 0) ok = wait(q_free, uint32_t(taken - 1) & 1u, p.status, 73);
            if (!ok) {
              ++t;
              break;
            }
            tc::mbar_arrive_expect_tx(q_full, L::kQ);
            for (int i = 0; i < HALVES; ++i) tma_load_5d(base + uint32_t(i * kTcRows * 128), &qmap, i * 64, 0, w.row0 / p.G, w.h, w.b, q_full);
            ++taken;
          }
        }
      }
      if (!ok) {  // copies that are on their way still land here
        for (int i = max(t - ST, 0); i < t; ++i) wait(k_full(i % ST), uint32_t(i / ST) & 1u, p.status, 63);
        for (int i = max(v_started - ST, 0); i < v_started; ++i) wait(v_full(i % ST), uint32_t(i / ST) & 1u, p.status, 63);
        if (taken > 0) wait(q_full, uint32_t(taken - 1) & 1u, p.status, 63);
      }
    }
  } else {
    // Tensor memory only behind the wait, and the next kernel only behind it: a block that held it while it waits could keep it from one that it
    // waits for.
    if (warp == 1) {
      tc::tmem_alloc(tc::smem_u32(tmem_at), 256);
      tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    asm volatile("bar.sync 1, 160;" ::: "memory");
    tc::fence_after_sync();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  const uint32_t tmem = warp == 0 ? 0u : *(volatile uint32_t*)tmem_at;

  if (warp == 1) {
    const uint32_t s_desc = tc::instr_desc(1, BF16 ? 1 : 0, kTcRows, kKeys), o_desc = tc::instr_desc(1, BF16 ? 1 : 0, kTcRows, HD) | (1u << 16);
    const uint32_t sum_desc = tc::instr_desc(1, BF16 ? 1 : 0, kTcRows, 16);
    const uint64_t ones = tc::smem_desc_sw128(base + L::kOnes);
    const bool one = tc::elect_one();
    bool ok = true;
    auto all_wait = [&](uint32_t b, uint32_t parity, unsigned site) { return bool(__all_sync(0xffffffffu, wait(b, parity, p.status, site))); };
    auto scores = [&](int t, bool last) {  // of the block's tile t, the last of its unit
      const int s = t % ST;
      if (!all_wait(k_full(s), uint32_t(t / ST) & 1u, 64)) return false;
      if (t > 0 && !all_wait(s_free, uint32_t(t - 1) & 1u, 67)) return false;
      tc::fence_after_sync();
      if (one) {
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          const uint64_t a = tc::smem_desc_sw128(base + uint32_t((x / 4) * kTcRows * 128 + (x % 4) * 32));
          const uint64_t k = tc::smem_desc_sw128(base + L::kK + uint32_t(s * L::kTile + (x / 4) * kKeys * 128 + (x % 4) * 32));
          tc::mma_f16(tmem, a, k, s_desc, x != 0);
        }
        tc::mma_commit(s_full);
        tc::mma_commit(k_free(s));
        if (last) tc::mma_commit(q_free);
      }
      __syncwarp();
      return true;
    };
    int t = 0, taken = 0;  // tiles and units with keys so far
    for (int u = int(blockIdx.x); u < p.units && ok; u += step) {
      const Unit w = unit(u);
      if (w.n == 0) continue;
      ok = all_wait(q_full, uint32_t(taken) & 1u, 71) && scores(t, w.n == 1);
      for (int j = 0; j < w.n && ok; ++j, ++t) {
        const int s = t % ST;
        if (j + 1 < w.n) ok = scores(t + 1, j + 2 == w.n);
        if (ok) ok = all_wait(v_full(s), uint32_t(t / ST) & 1u, 65);
        if (!ok) break;
        if (j == w.n - 1 && w.last_keys < kKeys) {  // values behind the last key may be anything, and their weights of zero would not silence a NaN
          const uint32_t v = base + L::kV + uint32_t(s * L::kTile);
          for (int x = 0; x < HALVES; ++x)
            for (int i = w.last_keys * 8 + lane; i < kKeys * 8; i += 32) tc::st_shared_v4(v + uint32_t(x * kKeys * 128 + i * 16), 0, 0, 0, 0);
          tc::fence_proxy_async_smem();
          __syncwarp();
        }
        if (j == 0 && taken > 0) ok = all_wait(o_free, uint32_t(taken - 1) & 1u, 72);
        if (ok) ok = all_wait(p_full, uint32_t(t) & 1u, 66);
        if (!ok) break;
        tc::fence_after_sync();
        if (one) {
#pragma unroll
          for (int x = 0; x < kKeys / 16; ++x) mma_f16_ts(tmem + kSum, tmem + kP + x * 8, ones, sum_desc, j != 0 || x != 0);
#pragma unroll
          for (int x = 0; x < kKeys / 16; ++x)
            mma_f16_ts(tmem + kOut, tmem + kP + x * 8, smem_desc_mn_sw128(base + L::kV + uint32_t(s * L::kTile + x * 2048), kKeys * 128), o_desc, j != 0 || x != 0);
          tc::mma_commit(o_done);
          tc::mma_commit(v_free(s));
        }
        __syncwarp();
      }
      ++taken;
    }
  } else if (warp >= 2) {
    const int quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t(quad * 32) << 16);
    bool ok = true;
    int t = 0;
    for (int u = int(blockIdx.x); u < p.units && ok; u += step) {
      const Unit w = unit(u);
      float m = -INFINITY;
      for (int j = 0; j < w.n; ++j, ++t) {
        ok = __all_sync(0xffffffffu, wait(s_full, uint32_t(t) & 1u, p.status, 68));
        if (!ok) break;
        tc::fence_after_sync();
        uint32_t s[kKeys / 32][32];
#pragma unroll
        for (int x = 0; x < kKeys / 32; ++x) tc::tmem_ld_32x32(lanes + x * 32, s[x]);
        tc::tmem_ld_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(s_free);
        if (j == w.n - 1 && w.last_keys < kKeys) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (i >= w.last_keys) s[i / 32][i % 32] = 0xff800000u;  // -inf
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kKeys; i += 2) mx[(i >> 1) & 1] = max3(mx[(i >> 1) & 1], __uint_as_float(s[i / 32][i % 32]), __uint_as_float(s[i / 32][i % 32 + 1]));
        const float high = fmaxf(mx[0], mx[1]) * p.scale_log2;
        // the weights' columns, and the result, are this warp's again when the product before is done
        if (j > 0) {
          ok = __all_sync(0xffffffffu, wait(o_done, uint32_t(t - 1) & 1u, p.status, 69));
          if (!ok) break;
          tc::fence_after_sync();
        }
        if (__any_sync(0xffffffffu, high > m + weight_growth(BF16))) {
          const float now = fmaxf(m, high);
          if (j > 0) {
            const float corr = m == now ? 1.f : ex2f(m - now);
            const float sum = __uint_as_float(tmem_ld_32x1(lanes + kSum));
            tc::tmem_ld_wait();
            tmem_st_32x1(lanes + kSum, __float_as_uint(sum * corr));
#pragma unroll
            for (int x = 0; x < HD / 16; ++x) {
              uint32_t o[16];
              tc::tmem_ld_32x16(lanes + kOut + x * 16, o);
              tc::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st_32x16(lanes + kOut + x * 16, o);
            }
          }
          m = now;
        }
        const float ref = m == -INFINITY ? 0.f : m - weight_lift(BF16);
        const unsigned long long scale2 = two(p.scale_log2, p.scale_log2), less2 = two(-ref, -ref);
#pragma unroll
        for (int x = 0; x < kKeys / 32; ++x) {
          uint32_t w16[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            unsigned long long v = two(__uint_as_float(s[x][2 * i]), __uint_as_float(s[x][2 * i + 1]));
            asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(v) : "l"(scale2), "l"(less2));
            if (i % 4 == 3) {
              v = ex2_poly(v);
            } else {
              float lo, hi;
              asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
              v = two(ex2f(lo), ex2f(hi));
            }
            float lo, hi;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
            w16[i] = pack16<BF16>(lo, hi);
          }
          tmem_st_32x16(lanes + kP + x * 16, w16);
        }
        tc::tmem_st_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full);
      }
      if (!ok) break;
      float sum = 0.f;
      if (w.n > 0) {
        ok = __all_sync(0xffffffffu, wait(o_done, uint32_t(t - 1) & 1u, p.status, 70));
        if (!ok) break;
        tc::fence_after_sync();
        sum = __uint_as_float(tmem_ld_32x1(lanes + kSum));
        tc::tmem_ld_wait();
      }
      if (m == -INFINITY && sum == sum) sum = 0.f;  // nothing above -inf
      const int rr = w.row0 + r, token = p.G == 1 ? rr : rr / p.G;
      const size_t place = size_t(max(w.rest, 0)) * p.part_rows + r;
      float* to = w.rest >= 0 ? p.parts + place * HD : nullptr;
      uint16_t* out = p.out + ((size_t(w.b) * p.R + token) * (p.Hkv * p.G) + w.h * p.G + rr - token * p.G) * HD;
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
      for (int x = 0; x < HD / 32; ++x) {
        uint32_t o[32];
        if (w.n > 0) {
          tc::tmem_ld_32x32(lanes + kOut + x * 32, o);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        if (x == HD / 32 - 1 && w.n > 0) {  // the next unit's products may overwrite it
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(o_free);
        }
        if (r < w.rows && to) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(to + x * 32 + i * 4) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else if (r < w.rows) {
          uint32_t w16[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w16[i] = pack16<BF16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(out + x * 32 + i * 8) = make_uint4(w16[4 * i], w16[4 * i + 1], w16[4 * i + 2], w16[4 * i + 3]);
        }
        __syncwarp();
      }
      if (to && r < w.rows) *reinterpret_cast<float2*>(p.stats + place * 2) = make_float2(m, sum);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) tc::tmem_dealloc(tmem, 256);
}

// The results of items that several blocks share: WARPS warps a row, 256 / (32 WARPS) rows a block.  The row's warps (half warps with 64 dimensions)
// take its parts in turn, all loads at once.  Two warps a row up to 16 parts, else eight
// (16 utterances of 224 rows on 1500 keys, the whole call in us: two 59.8, eight 66.8).
constexpr int kJoinThreads = 256;
// Volatile, or the compiler moves each load whose place it does not know to its use.
__device__ __forceinline__ float4 load_now(const float* p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}
// FULL: parts of 128 rows, at distances that the compiler knows (64 samples behind 45 000 keys: 55.9 us for 56.8)
template <int HD, bool BF16, int WARPS, bool FULL>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const float* parts, const float* stats, uint16_t* out, int n_parts, int rows_of_part, int first_item, int item_blocks, int tiles, int R, int G, int Hkv) {
  const int part_rows = FULL ? part_rows_of(kTcRows) : rows_of_part;
  constexpr int PER = HD / 4, TEAMS = 32 * WARPS / PER, ROWS = kJoinThreads / (32 * WARPS);  // threads of a part, parts at a time, rows
  constexpr int kMost = WARPS == 2 ? 16 : kMaxParts + 1;
  __shared__ float4 sums[ROWS][TEAMS][PER];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int in_block = int(threadIdx.x) / (32 * WARPS), thread = int(threadIdx.x) % (32 * WARPS);
  const int at = int(blockIdx.x) / item_blocks, r = int(blockIdx.x) % item_blocks * ROWS + in_block, item = first_item + at;
  const int rr = (item % tiles) * kTcRows + r;
  const bool there = rr < R * G;  // (else it reads what nobody wrote, or another row's, and writes nothing)
  const int lane = threadIdx.x & 31, team = thread / PER, e = (thread % PER) * 4;
  const size_t from = size_t(at) * n_parts * part_rows + min(r, part_rows - 1);  // the row's first part; the others part_rows on each
  const float *ml = behind_wait(stats + from * 2), *row = behind_wait(parts + from * HD + e);
  constexpr int kEach = (kMost + TEAMS - 1) / TEAMS, kLists = (kMost + 31) / 32;
  float4 o[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int x = i * TEAMS + team;
    if constexpr (FULL) o[i] = x < n_parts ? *reinterpret_cast<const float4*>(row + x * part_rows * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
    else o[i] = load_now(row + min(x, n_parts - 1) * part_rows * HD);  // (past the last: it again, not added)
  }
  // every warp: maxima and sums of all parts, two or three a lane
  float2 own[kLists];
  float mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kLists; ++i) {
    const int x = i * 32 + lane;
    own[i] = x < n_parts ? *reinterpret_cast<const float2*>(ml + x * part_rows * 2) : make_float2(-INFINITY, 0.f);
    mx = fmaxf(mx, own[i].x);
  }
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
#pragma unroll
  for (int i = 0; i < kLists; ++i) {
    const float w = own[i].y == 0.f ? 0.f : ex2f(own[i].x - mx);  // (a sum of NaN stays one)
    sum = fmaf(w, own[i].y, sum);
    own[i].x = w;
  }
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int x = i * TEAMS + team;  // its weight: with lane x % 32
    float w = 0.f;
#pragma unroll
    for (int j = 0; j < kLists; ++j) {
      const float v = __shfl_sync(0xffffffffu, own[j].x, x & 31);
      if (x / 32 == j) w = v;
    }
    if (x < n_parts) acc.x = fmaf(w, o[i].x, acc.x), acc.y = fmaf(w, o[i].y, acc.y), acc.z = fmaf(w, o[i].z, acc.z), acc.w = fmaf(w, o[i].w, acc.w);
  }
  sums[in_block][team][e / 4] = acc;
  __syncthreads();
  if (team != 0 || !there) return;
#pragma unroll
  for (int i = 1; i < TEAMS; ++i) {
    const float4 v = sums[in_block][i][e / 4];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int bh = item / tiles, h = bh % Hkv, b = bh / Hkv;
  *reinterpret_cast<uint2*>(out + ((size_t(b) * R + rr / G) * (Hkv * G) + h * G + rr % G) * HD + e) =
      make_uint2(pack16<BF16>(acc.x * inv, acc.y * inv), pack16<BF16>(acc.z * inv, acc.w * inv));
}

template <typename... Args>
int launch_behind(void (*kern)(Args...), int64_t blocks, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 0 : 1;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  return ASRQ_OK;
}

template <int HD, bool BF16>
int launch_flash(const CUtensorMap& qmap, const CUtensorMap& kmap, const CUtensorMap& vmap, const FlashParams& p, int sm_count, cudaStream_t stream) {
  auto kern = flash_kernel<HD, BF16>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), FlashLayout<HD>::kBytes);
  return rc ? rc : launch_behind(kern, std::min(p.units, 2 * sm_count), 192, FlashLayout<HD>::kBytes, stream, qmap, kmap, vmap, p);
}

}  // namespace

int rows_attention_join(const RowsParams& r, int hd, bool bf16, int64_t B, int64_t whole, const float* parts, const float* stats, int n_parts, cudaStream_t stream) {
  const int tiles = (r.R * r.G + kTcRows - 1) / kTcRows;
  const int64_t items = B * r.Hkv * tiles;
  if (whole >= items) return ASRQ_OK;
  const int part_rows = part_rows_of(int64_t(r.R) * r.G);
  auto go = [&](auto kern, int rows) {
    const int item_blocks = (std::min(r.R * r.G, kTcRows) + rows - 1) / rows;
    return launch_behind(kern, (items - whole) * item_blocks, kJoinThreads, 0, stream, parts, stats, r.out, n_parts, part_rows, int(whole), item_blocks, tiles, r.R, r.G, r.Hkv);
  };
  auto by_rows = [&](auto dim, auto type) {
    constexpr int HD = decltype(dim)::value;
    constexpr bool BF16 = decltype(type)::value;
    const bool full = part_rows == part_rows_of(kTcRows);
    if (n_parts <= 16) return full ? go(join_kernel<HD, BF16, 2, true>, 4) : go(join_kernel<HD, BF16, 2, false>, 4);
    return full ? go(join_kernel<HD, BF16, 8, true>, 1) : go(join_kernel<HD, BF16, 8, false>, 1);
  };
  if (hd == 64) return bf16 ? by_rows(std::integral_constant<int, 64>{}, std::true_type{}) : by_rows(std::integral_constant<int, 64>{}, std::false_type{});
  return bf16 ? by_rows(std::integral_constant<int, 128>{}, std::true_type{}) : by_rows(std::integral_constant<int, 128>{}, std::false_type{});
}

int rows_attention_tc(const RowsParams& r, int hd, bool bf16, int64_t B, const TcPlan& plan, float* parts, float* stats, int more, void* status, int sm_count, cudaStream_t stream) {
  FlashParams p = {};
  p.out = r.out, p.len = r.len;
  p.parts = parts, p.stats = stats;
  p.status = static_cast<unsigned*>(status);
  p.keys = r.keys;
  p.R = r.R, p.G = r.G, p.Hkv = r.Hkv;
  p.tiles = (r.R * r.G + kTcRows - 1) / kTcRows;
  p.whole = int(plan.whole);
  p.split = plan.split;
  p.slots = plan.split + more;
  p.part_rows = part_rows_of(int64_t(p.R) * p.G);
  p.scale_log2 = r.scale_log2;
  p.k_batch = r.k_b != 0, p.v_batch = r.v_b != 0, p.k_head = r.k_h != 0, p.v_head = r.v_h != 0;
  const uint32_t keys = hd == 64 ? FlashLayout<64>::kKeys : FlashLayout<128>::kKeys;
  CUtensorMap qmap, kmap, vmap;
  const TmapDim q_dims[4] = {{uint64_t(p.G), r.q_h, uint32_t(p.G)}, {uint64_t(p.R), r.q_r, uint32_t(kTcRows / p.G)}, {uint64_t(p.Hkv), p.G * r.q_h, 1}, {uint64_t(B), r.q_b, 1}};
  int rc = make_tmap_rows(&qmap, r.q, bf16, hd, 64, q_dims, 4);
  const TmapDim k_dims[3] = {{uint64_t(r.keys), r.k_t, keys}, {r.k_h ? uint64_t(r.Hkv) : 1, r.k_h, 1}, {r.k_b ? uint64_t(B) : 1, r.k_b, 1}};
  if (!rc) rc = make_tmap_rows(&kmap, r.k, bf16, hd, 64, k_dims, 3);
  const TmapDim v_dims[3] = {{uint64_t(r.keys), r.v_t, keys}, {r.v_h ? uint64_t(r.Hkv) : 1, r.v_h, 1}, {r.v_b ? uint64_t(B) : 1, r.v_b, 1}};
  if (!rc) rc = make_tmap_rows(&vmap, r.v, bf16, hd, 64, v_dims, 3);
  if (rc) return rc;
  p.units = int(plan.whole + (B * p.Hkv * p.tiles - plan.whole) * plan.split);
  if (hd == 64) return bf16 ? launch_flash<64, true>(qmap, kmap, vmap, p, sm_count, stream) : launch_flash<64, false>(qmap, kmap, vmap, p, sm_count, stream);
  return bf16 ? launch_flash<128, true>(qmap, kmap, vmap, p, sm_count, stream) : launch_flash<128, false>(qmap, kmap, vmap, p, sm_count, stream);
}

}  // namespace asrq
