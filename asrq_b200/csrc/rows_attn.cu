// Attention of several query rows of an utterance over keys that they share, with keys of their own behind them or not:
//
//   cross    the rows are the beams of a decoding step, or the tokens of a prompt, the keys an encoder's, each utterance's as many as it has;
//   prefix   the rows are beams or samples that share a prompt's keys; behind these each has its own.
//
// out[row] = sum_t w_t v_t / sum_t w_t, w_t = exp(scale q . k_t - m) over the row's keys, in one pass with the running maximum m
// and sum.  A row without keys is zero.  fp32 scores, softmax and accumulation.
//
// Bound: the bytes of the keys and values, read once for up to 16 rows (32 with heads of 64) of a key head.  A warp takes a chunk of
// 32 keys (16 with heads of 128) at a time, all dimensions, and keeps the rows' results in registers; the chunks of an item (utterance, key
// head, 16 rows) are dealt to the warps of a block or of a cluster of blocks, which meet at the end as (maximum, sum, values).
// Keys and values go from memory into the operands of mma.sync without passing shared memory, because a contraction may take its index
// in any order as long as both operands do, and so may the columns of the result:
//   scores   lane (g, c) of the operand holds dimensions 2c, 2c+1, 2c+8, 2c+9 of key g; it loads 16 consecutive bytes (dimensions 8c .. 8c+7 of 32) and
//            calls them the four pairs of two steps, for the queries alike;
//   values   the lane holds keys 2c, 2c+1, 2c+8, 2c+9 of column g: it loads 8 consecutive dimensions (8g ..) of each of the four keys, pairs the keys by a
//            byte permutation, and column g of tile j stands for dimension 8g + j.
// The next chunk's keys are loaded as soon as the scores are done, its values after the product.
#include <algorithm>
#include <type_traits>

#include "rows_attn.cuh"

namespace asrq {

int ensure_dynamic_smem(const void* kernel, size_t bytes);

namespace {

constexpr int kRowsWarps = 8;

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(u32_as_h2(w));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// behind the stream dependency, in program order; not kept in L1: a block reads it once
__device__ __forceinline__ uint4 ld_kv(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

template <int HD, int MT, bool BF16>
__global__ void __launch_bounds__(32 * kRowsWarps)
rows_attn_kernel(const __grid_constant__ RowsParams p) {
  constexpr int ROWS = 16 * MT;
  constexpr int KC = HD == 64 ? 32 : 16;              // keys of a chunk
  constexpr int NT = KC / 8, KS = HD / 16, DT = HD / 8;  // score tiles, steps of the scores, tiles of the result
  constexpr int PITCH = HD + 4;
  extern __shared__ __align__(16) float smem[];
  float* part = smem;                                  // warps x ROWS x PITCH: values, maximum, sum
  float* mine = smem + kRowsWarps * ROWS * PITCH;      // ROWS x PITCH: the block's
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, nw = blockDim.x >> 5;
  uint32_t rank, nsplit;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nsplit));
  const int item = int(blockIdx.x / nsplit);
  const int tile = item % p.tiles, bh = item / p.tiles, h = bh % p.Hkv, b = bh / p.Hkv;
  const int row0 = tile * ROWS, rows = min(ROWS, p.R * p.G - row0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // the row tile's chunks: the shared keys', then those of each of its rows' own keys, lane i holding the i-th's
  const long long n1 = p.len ? min(max(*(const volatile long long*)(p.len + b), 0ll), p.keys) : p.keys;
  const int chunks1 = int((n1 + KC - 1) / KC);
  const int first = row0 / p.G, n_own = p.k2 ? (row0 + rows - 1) / p.G - first + 1 : 0;
  long long len2 = 0;
  if (lane < n_own) len2 = min(max(*(const volatile long long*)(p.len2 + (p.len2_many ? (long long)b * p.R + first + lane : 0ll)), 0ll), p.keys2);
  const int chunks2 = int((len2 + KC - 1) / KC);
  int upto = chunks2;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  const int total = chunks1 + __shfl_sync(0xffffffffu, upto, 31);

  uint32_t qf[MT][KS][4];
  int own[MT][2];  // which of the tile's rows of `first` on a score row belongs to
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = row0 + mt * 16 + half * 8 + g;
      const bool there = r - row0 < rows;
      own[mt][half] = r / p.G - first;
      const uint16_t* src = p.q + b * p.q_b + (r / p.G) * p.q_r + (long long)(h * p.G + r % p.G) * p.q_h + c * 8;
#pragma unroll
      for (int ch = 0; ch < HD / 32; ++ch) {
        const uint4 u = there ? ld_x4(src + ch * 32) : make_uint4(0, 0, 0, 0);
        qf[mt][2 * ch][half] = u.x;
        qf[mt][2 * ch][2 + half] = u.y;
        qf[mt][2 * ch + 1][half] = u.z;
        qf[mt][2 * ch + 1][2 + half] = u.w;
      }
    }
  float o[MT][DT][4], m[MT][2], l[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt][0] = m[mt][1] = -INFINITY;
    l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < DT; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
  }

  struct Chunk {
    const uint16_t *k, *v;  // its first key
    long long kt, vt;
    int n, seg;             // keys there; -1: shared, else whose
  };
  auto chunk_at = [&](int i) {
    Chunk x;
    if (i < chunks1) {
      const long long t0 = (long long)i * KC;
      x.k = p.k + b * p.k_b + h * p.k_h + t0 * p.k_t;
      x.v = p.v + b * p.v_b + h * p.v_h + t0 * p.v_t;
      x.kt = p.k_t, x.vt = p.v_t;
      x.n = int(min(n1 - t0, (long long)KC));
      x.seg = -1;
    } else {
      const int s = __popc(__ballot_sync(0xffffffffu, upto <= i - chunks1));
      const long long t0 = (long long)(i - chunks1 - __shfl_sync(0xffffffffu, upto - chunks2, s)) * KC;
      const long long n = __shfl_sync(0xffffffffu, len2, s), r = (long long)b * p.R + first + s;
      x.k = p.k2 + r * p.k2_b + h * p.k2_h + t0 * p.k2_t;
      x.v = p.v2 + r * p.v2_b + h * p.v2_h + t0 * p.v2_t;
      x.kt = p.k2_t, x.vt = p.v2_t;
      x.n = int(min(n - t0, (long long)KC));
      x.seg = s;
    }
    return x;
  };
  uint4 kr[NT][HD / 32], vr[KC / 16][4][HD / 64];
  auto load_k = [&](const Chunk& x) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int t = j * 8 + g;
#pragma unroll
      for (int ch = 0; ch < HD / 32; ++ch) kr[j][ch] = t < x.n ? ld_kv(x.k + t * x.kt + ch * 32 + c * 8) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_v = [&](const Chunk& x) {
#pragma unroll
    for (int s = 0; s < KC / 16; ++s)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int t = s * 16 + (a >> 1) * 8 + 2 * c + (a & 1);
#pragma unroll
        for (int hh = 0; hh < HD / 64; ++hh) vr[s][a][hh] = t < x.n ? ld_kv(x.v + t * x.vt + hh * 64 + g * 8) : make_uint4(0, 0, 0, 0);
      }
  };
  const int step = int(nsplit) * nw;
  int at = int(rank) * nw + warp;
  Chunk cur, next;
  if (at < total) {
    cur = chunk_at(at);
    load_k(cur);
    load_v(cur);
  }
#pragma unroll 1
  for (; at < total; at += step) {
    const bool more = at + step < total;
    if (more) next = chunk_at(at + step);
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
#pragma unroll
        for (int ch = 0; ch < HD / 32; ++ch) {
          mma16816<BF16>(s[mt][j], qf[mt][2 * ch], kr[j][ch].x, kr[j][ch].y);
          mma16816<BF16>(s[mt][j], qf[mt][2 * ch + 1], kr[j][ch].z, kr[j][ch].w);
        }
      }
    if (more) load_k(next);
    uint32_t pr[MT][NT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool live = j * 8 + 2 * c + (e & 1) < cur.n && (cur.seg < 0 || cur.seg == own[mt][e >> 1]);
          s[mt][j][e] = live ? s[mt][j][e] * p.scale_log2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[mt][j][e]);
        }
      float base[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
        const float now = fmaxf(m[mt][half], mx[half]);
        base[half] = now == -INFINITY ? 0.f : now;  // no key of this row yet
        const float corr = ex2(m[mt][half] - base[half]);
        m[mt][half] = now;
        l[mt][half] *= corr;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
          o[mt][j][2 * half] *= corr;
          o[mt][j][2 * half + 1] *= corr;
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float a = ex2(s[mt][j][2 * half] - base[half]), d = ex2(s[mt][j][2 * half + 1] - base[half]);
          pr[mt][j][half] = pack2<BF16>(a, d);
          const float2 r = unpack2<BF16>(pr[mt][j][half]);  // the sum is that of the rounded weights
          l[mt][half] += r.x + r.y;
        }
    }
    // Own keys are those of some rows only: the others' weights are zero, but a zero times an infinity is not, so their results stay out.
    auto product = [&](auto shared) {
#pragma unroll
      for (int hh = 0; hh < HD / 64; ++hh)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const int j = hh * 8 + 2 * w + odd;
            float add[MT][4] = {};
#pragma unroll
            for (int st = 0; st < KC / 16; ++st) {
              auto word = [&](int a) { return w == 0 ? vr[st][a][hh].x : w == 1 ? vr[st][a][hh].y : w == 2 ? vr[st][a][hh].z : vr[st][a][hh].w; };
              const uint32_t b0 = prmt(word(0), word(1), odd ? 0x7632u : 0x5410u), b1 = prmt(word(2), word(3), odd ? 0x7632u : 0x5410u);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                const uint32_t a[4] = {pr[mt][2 * st][0], pr[mt][2 * st][1], pr[mt][2 * st + 1][0], pr[mt][2 * st + 1][1]};
                mma16816<BF16>(shared.value ? o[mt][j] : add[mt], a, b0, b1);
              }
            }
            if (!shared.value) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (cur.seg == own[mt][e >> 1]) o[mt][j][e] += add[mt][e];
            }
          }
    };
    if (cur.seg < 0) product(std::true_type{});
    else product(std::false_type{});
    if (more) load_v(next);
    cur = next;
  }
  // the warps' parts, the block's, the cluster's
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 1);
      l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 2);
      const int r = mt * 16 + half * 8 + g;
      if (r >= rows) continue;
      float* d = part + (warp * ROWS + r) * PITCH;
#pragma unroll
      for (int hh = 0; hh < HD / 64; ++hh)
#pragma unroll
        for (int e = 0; e < 2; ++e)  // columns 2c and 2c + 1 of the tiles: dimensions 16c .. and 16c + 8 ..
#pragma unroll
          for (int q4 = 0; q4 < 2; ++q4) {
            const int j = hh * 8 + q4 * 4, x = 2 * half + e;
            *reinterpret_cast<float4*>(d + hh * 64 + 16 * c + 8 * e + 4 * q4) = make_float4(o[mt][j][x], o[mt][j + 1][x], o[mt][j + 2][x], o[mt][j + 3][x]);
          }
      if (c == 0) {
        d[HD] = m[mt][half];
        d[HD + 1] = l[mt][half];
      }
    }
  __syncthreads();
  const int Hq = p.Hkv * p.G;
  auto put = [&](int r, int e, float v, float sum) {  // element e of the tile's row r
    const int rr = row0 + r;
    p.out[((size_t(b) * p.R + rr / p.G) * Hq + h * p.G + rr % p.G) * HD + e] = float_to_out16(sum > 0.f || sum != sum ? v / sum : 0.f, BF16);
  };
  for (int i = threadIdx.x; i < rows * HD; i += blockDim.x) {
    const int r = i / HD, e = i % HD;
    float mx = -INFINITY, acc = 0.f, sum = 0.f;
    for (int w = 0; w < nw; ++w) mx = fmaxf(mx, part[(w * ROWS + r) * PITCH + HD]);
    const int n_parts = rank == 0 ? p.n_parts : 0, rr = row0 + r;  // what the tensor-core kernel left
    const float* from = p.parts + (size_t(bh) * ((p.R * p.G + kTcRows - 1) / kTcRows) + rr / kTcRows) * p.n_parts * part_floats(HD);
    const int row_at = (rr % kTcRows) * HD + e, ml_at = kTcRows * HD + (rr % kTcRows) * 2;
    for (int x = 0; x < n_parts; ++x) mx = fmaxf(mx, from[size_t(x) * part_floats(HD) + ml_at]);
#pragma unroll 4
    for (int x = 0; x < n_parts; ++x) {
      const float* d = from + size_t(x) * part_floats(HD);
      const float wt = d[ml_at + 1] == 0.f ? 0.f : ex2(d[ml_at] - mx);
      acc = fmaf(wt, d[row_at], acc);
      sum = fmaf(wt, d[ml_at + 1], sum);
    }
    for (int w = 0; w < nw; ++w) {
      const float* d = part + (w * ROWS + r) * PITCH;
      const float wt = d[HD + 1] == 0.f ? 0.f : ex2(d[HD] - mx);  // a sum of NaN stays one
      acc = fmaf(wt, d[e], acc);
      sum = fmaf(wt, d[HD + 1], sum);
    }
    if (nsplit == 1) {
      put(r, e, acc, sum);
    } else {
      mine[r * PITCH + e] = acc;
      if (e == 0) {
        mine[r * PITCH + HD] = mx;
        mine[r * PITCH + HD + 1] = sum;
      }
    }
  }
  if (nsplit == 1) return;
  tc::cluster_sync();  // every block's part is there
  const uint32_t base = tc::smem_u32(mine);
  for (int i = int(rank) * int(blockDim.x) + threadIdx.x; i < rows * HD; i += int(nsplit) * int(blockDim.x)) {
    const int r = i / HD, e = i % HD;
    float mx = -INFINITY, acc = 0.f, sum = 0.f;
    for (uint32_t x = 0; x < nsplit; ++x) mx = fmaxf(mx, tc::ld_dsmem_f32(tc::mapa(base + uint32_t(r * PITCH + HD) * 4u, x)));
    for (uint32_t x = 0; x < nsplit; ++x) {
      const uint32_t d = tc::mapa(base + uint32_t(r * PITCH) * 4u, x);
      const float part_sum = tc::ld_dsmem_f32(d + HD * 4u + 4u), wt = part_sum == 0.f ? 0.f : ex2(tc::ld_dsmem_f32(d + HD * 4u) - mx);
      acc = fmaf(wt, tc::ld_dsmem_f32(d + uint32_t(e) * 4u), acc);
      sum = fmaf(wt, part_sum, sum);
    }
    put(r, e, acc, sum);
  }
  tc::cluster_sync();  // none leaves while another reads its part
}

template <int HD, int MT, bool BF16>
int launch_rows(RowsParams p, int64_t B, int sm_count, cudaStream_t stream) {
  constexpr int ROWS = 16 * MT, KC = HD == 64 ? 32 : 16;
  constexpr size_t smem = size_t(kRowsWarps + 1) * ROWS * (HD + 4) * 4;
  p.tiles = (p.R * p.G + ROWS - 1) / ROWS;
  const int64_t items = B * p.Hkv * p.tiles;
  auto kern = rows_attn_kernel<HD, MT, BF16>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (rc) return rc;
  // blocks an item: until the chip is full, or a warp has a single chunk
  const int64_t chunks = (p.keys + KC - 1) / KC + (p.k2 ? (p.keys2 + KC - 1) / KC : 0);
  int split = 1;
  while (split < 8 && items * split * 2 <= sm_count * 5 / 4 && chunks > split * kRowsWarps) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(items * split));
  cfg.blockDim = dim3(32 * kRowsWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(kOptNoPdl) ? 1 : 2;
  ASRQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  return ASRQ_OK;
}

}  // namespace

// Whether the tensor-core kernel takes a call, and the parts it divides the keys into (0: it does not).
// @RULE
int tc_parts(int64_t B, int64_t R, int G, int n_kv_heads, int hd, int64_t keys, bool own, int sm_count) {
  const int64_t rows = R * G, tiles = (rows + kTcRows - 1) / kTcRows, items = B * n_kv_heads * tiles, key_tiles = (keys + 63) / 64;
  if (rows <= (hd == 64 ? 32 : 16) || keys < 64) return 0;
  const int64_t slots = 2 * sm_count;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 64 && (s == 1 || key_tiles / s >= 4); ++s) {
    const int64_t cost = (items * s + slots - 1) / slots * ((key_tiles + s - 1) / s + 4) + (s > 1 || own ? 4 + items * s * tiles / slots : 0);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

size_t rows_attention_scratch_bytes(int64_t B, int64_t R, int n_q_heads, int n_kv_heads, int hd, int64_t keys, int64_t keys2, int sm_count) {
  const int G = n_q_heads / n_kv_heads, n = tc_parts(B, R, G, n_kv_heads, hd, keys, keys2 > 0, sm_count);
  if (n == 0 || (n == 1 && keys2 == 0)) return 0;
  return size_t(B) * n_kv_heads * ((R * G + kTcRows - 1) / kTcRows) * n * part_floats(hd) * sizeof(float);
}

int rows_attention(const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v, const int64_t* vs, const long long* lengths,
                   const void* k2, const int64_t* k2s, const void* v2, const int64_t* v2s, const long long* lengths2, bool lengths2_many, void* out,
                   int64_t B, int64_t R, int n_q_heads, int n_kv_heads, int hd, int64_t keys, int64_t keys2, float scale, int dtype, void* status, void* scratch,
                   size_t scratch_bytes, int sm_count, cudaStream_t stream) {
  RowsParams p = {};
  auto in = [](const void* x) { return static_cast<const uint16_t*>(x); };
  p.q = in(q), p.q_b = qs[0], p.q_r = qs[1], p.q_h = qs[2];
  p.out = static_cast<uint16_t*>(out);
  p.k = in(k), p.k_b = ks[0], p.k_h = ks[1], p.k_t = ks[2];
  p.v = in(v), p.v_b = vs[0], p.v_h = vs[1], p.v_t = vs[2];
  p.len = lengths;
  p.keys = keys;
  if (k2) {
    p.k2 = in(k2), p.k2_b = k2s[0], p.k2_h = k2s[1], p.k2_t = k2s[2];
    p.v2 = in(v2), p.v2_b = v2s[0], p.v2_h = v2s[1], p.v2_t = v2s[2];
    p.len2 = lengths2;
    p.len2_many = lengths2_many;
    p.keys2 = keys2;
  }
  p.R = int(R), p.G = n_q_heads / n_kv_heads, p.Hkv = n_kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  const bool bf16 = dtype == ASRQ_BF16;
  int parts = status && ((ks[2] && vs[2]) || keys == 1) ? tc_parts(B, R, p.G, n_kv_heads, hd, keys, k2 != nullptr, sm_count) : 0;
  if (parts > 0) {
    const size_t part_bytes = size_t(B) * n_kv_heads * ((R * p.G + kTcRows - 1) / kTcRows) * part_floats(hd) * sizeof(float);
    const bool kept = scratch && scratch_bytes >= part_bytes * parts;
    if (!kept && !k2) parts = 1;
    if (kept || !k2) {
      const bool direct = parts == 1 && !k2;
      const int rc = rows_attention_tc(p, hd, bf16, B, parts, direct ? nullptr : static_cast<float*>(scratch), status, sm_count, stream);
      if (rc || direct) return rc;
      p.parts = static_cast<const float*>(scratch);
      p.n_parts = parts;
      p.keys = 0;
    }
  }
  if (hd == 128) return bf16 ? launch_rows<128, 1, true>(p, B, sm_count, stream) : launch_rows<128, 1, false>(p, B, sm_count, stream);
  if (R * p.G > 16) return bf16 ? launch_rows<64, 2, true>(p, B, sm_count, stream) : launch_rows<64, 2, false>(p, B, sm_count, stream);
  return bf16 ? launch_rows<64, 1, true>(p, B, sm_count, stream) : launch_rows<64, 1, false>(p, B, sm_count, stream);
}

}  // namespace asrq
