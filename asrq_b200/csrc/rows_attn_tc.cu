// Attention of many query rows over keys that they share, on the 5th-generation tensor cores: the tokens of a prompt over an encoder's
// states, or the rows of many beams or samples over their prompt.
//
// A block holds 128 rows (all query heads of a key head, so several tokens or beams) and walks its keys 64 at a time: S = Q K^T into tensor
// memory, a thread per row reads its 64 scores, and writes the weights 2^(scale' s - m) back over them in 16 bits, from where
// O += P V takes them as its first operand.  K arrives by TMA as rows of the contraction, V as it lies, dimensions contiguous, which the
// second operand's descriptor calls MN-major.  Two score buffers: S of the next keys is done while these are exponentiated; two blocks an
// SM fill each other's waits.
// The reference exponent m of a row moves only when its maximum has grown by more than 8 (a weight stays below 2^8, a sum in 32 bits has
// room for that): O is scaled at the first tiles and hardly ever after.
//
// Bound: at 64 dimensions the exponentials, 16 a cycle and SM; at 128 these and the memory's bytes where few rows share many keys.
#include "rows_attn.cuh"

namespace asrq {

int ensure_dynamic_smem(const void* kernel, size_t bytes);

namespace {

constexpr int kKeys = 64;  // of a tile

struct FlashParams {
  const uint16_t* q;
  uint16_t* out;
  const long long* len;
  float* parts;
  unsigned* status;
  long long q_b, q_r, q_h, keys;
  int R, G, Hkv, tiles, split, k_batch, v_batch, k_head, v_head;  // *_batch, *_head: 0 where all utterances or heads share them
  float scale_log2;  // not negative
  uint32_t q_flip;   // the sign bits of a query pair where the scale is
};

template <int HD>
struct FlashLayout {
  static constexpr int kStages = HD == 64 ? 4 : 2;
  static constexpr int kQ = kTcRows * HD * 2, kTile = kKeys * HD * 2;
  static constexpr int kK = kQ, kV = kQ + kStages * kTile, kBars = kQ + 2 * kStages * kTile;
  static constexpr int kBytes = kBars + (4 * kStages + 5) * 8 + 16 + 1024;  // 1024: the base is aligned to it
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
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

template <int HD, bool BF16>
__global__ void __launch_bounds__(192, 2)
flash_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ FlashParams p) {
  using L = FlashLayout<HD>;
  constexpr int ST = L::kStages, HALVES = HD / 64;
  constexpr uint32_t kOut = 128;  // tensor memory: two score buffers of 64 columns, then the result
  extern __shared__ uint8_t flash_smem[];
  const uint32_t base = (tc::smem_u32(flash_smem) + 1023u) & ~1023u;
  uint8_t* smem = flash_smem + (base - tc::smem_u32(flash_smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [&](int i) { return base + L::kBars + uint32_t(i) * 8u; };
  auto k_full = [&](int s) { return bar(s); };
  auto k_free = [&](int s) { return bar(ST + s); };
  auto v_full = [&](int s) { return bar(2 * ST + s); };
  auto v_free = [&](int s) { return bar(3 * ST + s); };
  auto s_full = [&](int i) { return bar(4 * ST + i); };
  auto p_full = [&](int i) { return bar(4 * ST + 2 + i); };
  const uint32_t o_done = bar(4 * ST + 4);
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + L::kBars + (4 * ST + 5) * 8);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 4 * ST + 2; ++i) tc::mbar_init(bar(i), 1);
    tc::mbar_init(p_full(0), 4);
    tc::mbar_init(p_full(1), 4);
    tc::mbar_init(o_done, 1);
    tc::fence_barrier_init();
    tc::prefetch_tmap(&kmap);
    tc::prefetch_tmap(&vmap);
  }
  const int part = int(blockIdx.x % unsigned(p.split)), item = int(blockIdx.x / unsigned(p.split));
  const int tile = item % p.tiles, bh = item / p.tiles, h = bh % p.Hkv, b = bh / p.Hkv;
  const int row0 = tile * kTcRows, rows = min(kTcRows, p.R * p.G - row0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // Tensor memory only now, and the next kernel only behind it: a block that held it while it waits could keep it from one that it waits for.
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(tmem_at), 256);
    tc::tmem_relinquish();
  }
  const long long n_keys = p.len ? min(max(*(const volatile long long*)(p.len + b), 0ll), p.keys) : p.keys;
  const int all = int((n_keys + kKeys - 1) / kKeys), t0 = int((long long)all * part / p.split), n = int((long long)all * (part + 1) / p.split) - t0;
  const int last_keys = t0 + n == all ? int(n_keys - (long long)(all - 1) * kKeys) : kKeys;  // of this block's last tile

  // Q, rows of the contraction, 64 dimensions (128 bytes, chunks of 16 exchanged by the row) at a time
  for (int i = threadIdx.x; i < kTcRows * HD / 8; i += 192) {
    const int r = i / (HD / 8), c = i % (HD / 8), rr = row0 + r;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (r < rows) u = ld_x4(p.q + b * p.q_b + (rr / p.G) * p.q_r + (long long)(h * p.G + rr % p.G) * p.q_h + c * 8);
    u.x ^= p.q_flip, u.y ^= p.q_flip, u.z ^= p.q_flip, u.w ^= p.q_flip;
    tc::st_shared_v4(base + uint32_t((c / 8) * kTcRows * 128 + r * 128 + (((c % 8) ^ (r & 7)) * 16)), u.x, u.y, u.z, u.w);
  }
  tc::fence_proxy_async_smem();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *(volatile uint32_t*)tmem_at;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      const int kb = p.k_batch ? b : 0, kh = p.k_head ? h : 0, vb = p.v_batch ? b : 0, vh = p.v_head ? h : 0;
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const int s = j % ST;
        const uint32_t ph = uint32_t(j / ST) & 1u;
        ok = tc::mbar_wait(k_free(s), ph ^ 1u, p.status, 61);
        if (!ok) break;
        tc::mbar_arrive_expect_tx(k_full(s), L::kTile);
        for (int x = 0; x < HALVES; ++x) tma_load_4d(base + L::kK + uint32_t(s * L::kTile + x * kKeys * 128), &kmap, x * 64, (t0 + j) * kKeys, kh, kb, k_full(s));
        ok = tc::mbar_wait(v_free(s), ph ^ 1u, p.status, 62);
        if (!ok) break;
        tc::mbar_arrive_expect_tx(v_full(s), L::kTile);
        for (int x = 0; x < HALVES; ++x) tma_load_4d(base + L::kV + uint32_t(s * L::kTile + x * kKeys * 128), &vmap, x * 64, (t0 + j) * kKeys, vh, vb, v_full(s));
      }
      if (!ok)  // copies that are on their way still land here
        for (int s = 0; s < ST; ++s) {
          tc::mbar_wait(k_full(s), 0, p.status, 63);
          tc::mbar_wait(v_full(s), 0, p.status, 63);
        }
    }
  } else if (warp == 1) {
    const uint32_t s_desc = tc::instr_desc(1, BF16 ? 1 : 0, kTcRows, kKeys), o_desc = tc::instr_desc(1, BF16 ? 1 : 0, kTcRows, HD) | (1u << 16);
    const bool one = tc::elect_one();
    bool ok = true;
    auto scores = [&](int j) {  // of tile j
      const int s = j % ST;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(k_full(s), uint32_t(j / ST) & 1u, p.status, 64))) return false;
      tc::fence_after_sync();
      if (one) {
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          const uint64_t a = tc::smem_desc_sw128(base + uint32_t((x / 4) * kTcRows * 128 + (x % 4) * 32));
          const uint64_t k = tc::smem_desc_sw128(base + L::kK + uint32_t(s * L::kTile + (x / 4) * kKeys * 128 + (x % 4) * 32));
          tc::mma_f16(tmem + uint32_t(j & 1) * kKeys, a, k, s_desc, x != 0);
        }
        tc::mma_commit(s_full(j & 1));
        tc::mma_commit(k_free(s));
      }
      __syncwarp();
      return true;
    };
    for (int j = 0; j < min(n, 2) && ok; ++j) ok = scores(j);
    for (int j = 0; j < n && ok; ++j) {
      const int s = j % ST;
      ok = __all_sync(0xffffffffu, tc::mbar_wait(v_full(s), uint32_t(j / ST) & 1u, p.status, 65));
      if (!ok) break;
      if (j == n - 1 && last_keys < kKeys) {  // values behind the last key may be anything, and their weights of zero would not silence a NaN
        const uint32_t v = base + L::kV + uint32_t(s * L::kTile);
        for (int x = 0; x < HALVES; ++x)
          for (int i = last_keys * 8 + lane; i < kKeys * 8; i += 32) tc::st_shared_v4(v + uint32_t(x * kKeys * 128 + i * 16), 0, 0, 0, 0);
        tc::fence_proxy_async_smem();
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, tc::mbar_wait(p_full(j & 1), uint32_t(j >> 1) & 1u, p.status, 66));
      if (!ok) break;
      tc::fence_after_sync();
      if (one) {
#pragma unroll
        for (int x = 0; x < kKeys / 16; ++x)
          mma_f16_ts(tmem + kOut, tmem + uint32_t(j & 1) * kKeys + x * 8, smem_desc_mn_sw128(base + L::kV + uint32_t(s * L::kTile + x * 2048), kKeys * 128), o_desc,
                     j != 0 || x != 0);
        tc::mma_commit(o_done);
        tc::mma_commit(v_free(s));
      }
      __syncwarp();
      if (j + 2 < n) {  // its scores go where these weights were read
        ok = __all_sync(0xffffffffu, tc::mbar_wait(o_done, uint32_t(j) & 1u, p.status, 67));
        if (ok) ok = scores(j + 2);
      }
    }
  } else {
    const int quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t(quad * 32) << 16);
    float m = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = __all_sync(0xffffffffu, tc::mbar_wait(s_full(j & 1), uint32_t(j >> 1) & 1u, p.status, 68));
      if (!ok) break;
      tc::fence_after_sync();
      uint32_t s[2][32];
      const uint32_t at = lanes + uint32_t(j & 1) * kKeys;
      tc::tmem_ld_32x32(at, s[0]);
      tc::tmem_ld_32x32(at + 32, s[1]);
      tc::tmem_ld_wait();
      if (j == n - 1 && last_keys < kKeys) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (i >= last_keys) s[i / 32][i % 32] = 0xff800000u;  // -inf
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kKeys; ++i) mx[i % 4] = fmaxf(mx[i % 4], __uint_as_float(s[i / 32][i % 32]));
      const float high = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      if (__any_sync(0xffffffffu, high > m + 8.f)) {
        const float now = fmaxf(m, high);
        if (j > 0) {
          ok = __all_sync(0xffffffffu, tc::mbar_wait(o_done, uint32_t(j - 1) & 1u, p.status, 69));
          if (!ok) break;
          tc::fence_after_sync();
          const float corr = m == now ? 1.f : ex2f(m - now);
          sum *= corr;
#pragma unroll
          for (int x = 0; x < HD / 32; ++x) {
            uint32_t o[32];
            tc::tmem_ld_32x32(lanes + kOut + x * 32, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tc::tmem_st_32x32(lanes + kOut + x * 32, o);
          }
        }
        m = now;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      const unsigned long long scale2 = two(p.scale_log2, p.scale_log2), less2 = two(-ref, -ref);
      unsigned long long acc[2] = {0, 0};
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        unsigned long long x = two(__uint_as_float(s[i / 16][(2 * i) % 32]), __uint_as_float(s[i / 16][(2 * i + 1) % 32]));
        asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(x) : "l"(scale2), "l"(less2));
        float lo, hi;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
        lo = ex2f(lo);
        hi = ex2f(hi);
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc[i % 2]) : "l"(two(lo, hi)));
        w[i] = pack16<BF16>(lo, hi);
      }
      asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc[0]) : "l"(acc[1]));
      float a0, a1;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(acc[0]));
      sum += a0 + a1;
      tc::tmem_st_32x32(at, w);
      tc::tmem_st_wait();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full(j & 1));
    }
    // (the product before the last one may not be done either, and its phase is the one that would be taken for the last's)
    for (int j = max(n - 2, 0); j < n && ok; ++j) ok = __all_sync(0xffffffffu, tc::mbar_wait(o_done, uint32_t(j) & 1u, p.status, 70));
    tc::fence_after_sync();
    const int rr = row0 + r;
    float* to = p.parts ? p.parts + size_t(blockIdx.x) * part_floats(HD) : nullptr;
    uint16_t* out = p.out + ((size_t(b) * p.R + rr / p.G) * (p.Hkv * p.G) + h * p.G + rr % p.G) * HD;
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int x = 0; x < HD / 32; ++x) {
      uint32_t o[32];
      if (n > 0 && ok) {
        tc::tmem_ld_32x32(lanes + kOut + x * 32, o);
        tc::tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0;
      }
      if (r < rows && to) {
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(to + r * HD + x * 32 + i * 4) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else if (r < rows) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pack16<BF16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(out + x * 32 + i * 8) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
      __syncwarp();
    }
    if (to && r < rows) *reinterpret_cast<float2*>(to + kTcRows * HD + r * 2) = make_float2(m, sum);
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) tc::tmem_dealloc(tmem, 256);
}

template <int HD, bool BF16>
int launch_flash(const CUtensorMap& kmap, const CUtensorMap& vmap, const FlashParams& p, int64_t blocks, cudaStream_t stream) {
  auto kern = flash_kernel<HD, BF16>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), FlashLayout<HD>::kBytes);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = FlashLayout<HD>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 0 : 1;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, kmap, vmap, p));
  return ASRQ_OK;
}

}  // namespace

int rows_attention_tc(const RowsParams& r, int hd, bool bf16, int64_t B, int n_parts, float* parts, void* status, int sm_count, cudaStream_t stream) {
  FlashParams p = {};
  p.q = r.q, p.out = r.out, p.len = r.len;
  p.parts = parts;
  p.status = static_cast<unsigned*>(status);
  p.q_b = r.q_b, p.q_r = r.q_r, p.q_h = r.q_h, p.keys = r.keys;
  p.R = r.R, p.G = r.G, p.Hkv = r.Hkv;
  p.tiles = (r.R * r.G + kTcRows - 1) / kTcRows;
  p.split = n_parts;
  p.scale_log2 = r.scale_log2 < 0.f ? -r.scale_log2 : r.scale_log2;
  p.q_flip = r.scale_log2 < 0.f ? 0x80008000u : 0u;
  p.k_batch = r.k_b != 0, p.v_batch = r.v_b != 0, p.k_head = r.k_h != 0, p.v_head = r.v_h != 0;
  CUtensorMap kmap, vmap;
  int rc = make_tmap_4d(&kmap, r.k, bf16, hd, uint64_t(r.keys), r.k_h ? r.Hkv : 1, r.k_b ? uint64_t(B) : 1, r.k_t, r.k_h, r.k_b, 64, kKeys);
  if (!rc) rc = make_tmap_4d(&vmap, r.v, bf16, hd, uint64_t(r.keys), r.v_h ? r.Hkv : 1, r.v_b ? uint64_t(B) : 1, r.v_t, r.v_h, r.v_b, 64, kKeys);
  if (rc) return rc;
  const int64_t blocks = B * p.Hkv * p.tiles * n_parts;
  if (hd == 64) return bf16 ? launch_flash<64, true>(kmap, vmap, p, blocks, stream) : launch_flash<64, false>(kmap, vmap, p, blocks, stream);
  return bf16 ? launch_flash<128, true>(kmap, vmap, p, blocks, stream) : launch_flash<128, false>(kmap, vmap, p, blocks, stream);
}

}  // namespace asrq
