// Attention of several query rows of an utterance over keys that they share, with keys of their own behind them or not:
//
//   cross    the rows are the beams of a decoding step, or the tokens of a prompt, the keys an encoder's, each utterance's as many as it has;
//   prefix   the rows are beams or samples that share a prompt's keys; behind these each has its own.
//
// out[row] = sum_t w_t v_t / sum_t w_t, w_t = exp(scale q . k_t - m) over the row's keys, in one pass with the running maximum m
// and sum.  A row without keys is zero.  fp32 scores, softmax and accumulation; the weights are rounded to the values' type, which the second product
// takes, and the sum is that of the rounded ones.
//
// Bound: the bytes of the keys and values, read once for up to 16 rows (32 with heads of 64) of a key head.  A warp takes a chunk of
// 32 keys (16 with heads of 128) at a time, all dimensions, and keeps the rows' results in registers; the chunks of an item (utterance, key
// head, 16 rows) are dealt to the warps of a block or of a cluster of blocks, which meet at the end as (maximum, sum, values).
// Each warp has two chunks of 8 KB in shared memory and copies for itself, one ahead, with no block-wide wait until the end: 32 utterances of 5 rows
// on 1500 keys take 42 us, 5.9 TB/s (66 us with the chunks in registers; 50 with three chunks and fewer warps).  Many items are bound by the
// waves they come in, one utterance by latency: 5.4 us for 5 rows on 1500 keys.  A contraction may take its index in any order as long as both operands do, and so may the
// columns of the result, so that lanes read 16 bytes of a key at a time: lane (g, c) of the operand holds dimensions 2c, 2c+1, 2c+8, 2c+9 of
// key g; it reads 16 consecutive bytes (dimensions 8c .. 8c+7 of 32) and calls them the four pairs of two steps, for the queries alike.  Values
// are turned on their way by ldmatrix.  The 16-byte pieces of a key lie exchanged so that the eight lanes of a read meet all banks: by 4 in
// odd keys, those of values by the key.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cluster_choice.h"
#include "rows_attn.cuh"

namespace asrq {

int ensure_dynamic_smem(const void* kernel, size_t bytes);

namespace {

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
__device__ __forceinline__ void copy16(uint32_t to, const uint16_t* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t to, const uint16_t* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
// four 8 x 8 matrices of 16-bit values, rows at the lanes' addresses, each turned over
__device__ __forceinline__ void ldmatrix_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// acc + v * 0 of a pair: stays zero but for infinities and NaN
template <bool BF16>
__device__ __forceinline__ uint32_t times_zero(uint32_t v, uint32_t acc) {
  uint32_t r;
  if constexpr (BF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0u), "r"(acc));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0u), "r"(acc));
  return r;
}
constexpr int kStages = 2, kChunkBytes = 8192;  // a warp's: keys, then values

template <int HD, int MT, bool BF16>
__global__ void __launch_bounds__(32 * kRowsWarps) __maxnreg__(MT == 1 ? 168 : 240)
rows_attn_kernel(const __grid_constant__ RowsParams p) {
  constexpr int ROWS = 16 * MT;
  constexpr int KC = HD == 64 ? 32 : 16;              // keys of a chunk
  constexpr int NT = KC / 8, KS = HD / 16, DT = HD / 8;  // score tiles, steps of the scores, tiles of the result
  constexpr int PITCH = HD + 4;
  extern __shared__ __align__(16) float smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, nw = blockDim.x >> 5;
  constexpr int kPart = kStages * kChunkBytes / 4;  // floats from a warp's part to the next: they lie over the chunks
  static_assert(ROWS * PITCH <= kPart, "a part fits");
  float* part = smem;                        // of each warp ROWS x PITCH: values, maximum, sum; the sums become weights
  float* gathered = part + nw * kPart;       // ROWS x HD: this block's share of the result, from every block of the cluster
  float* stats = gathered + ROWS * HD;       // blocks x ROWS x 2: their maxima and sums
  float* total_of = stats + 2 * kMaxSplit * ROWS;  // ROWS x 2: the block's (then the cluster's) maximum and sum
  uint32_t rank, nsplit;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nsplit));
  // a block's shared memory may be written by another only once it is known to run: arrived here, waited for before the first write
  if (nsplit > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int item = int(blockIdx.x / nsplit);
  const int tile = item % p.tiles, bh = item / p.tiles, h = bh % p.Hkv, b = bh / p.Hkv;
  const int row0 = tile * ROWS, rows = min(ROWS, p.R * p.G - row0);
  // Behind the tensor-core kernel of the same call, which has itself waited for all before it, nothing is waited for until the end.
  if (!p.parts) asm volatile("griddepcontrol.wait;" ::: "memory");
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

  const uint32_t mem = tc::smem_u32(smem) + uint32_t(warp * kStages * kChunkBytes);
  constexpr int PER = HD / 8, EACH = 32 / PER;  // pieces of a key; keys the warp's lanes copy at a time
  const int copy_t = lane / PER, copy_piece = lane % PER;
  const uint16_t *k1 = p.k + b * p.k_b + h * p.k_h + copy_t * p.k_t + copy_piece * 8, *v1 = p.v + b * p.v_b + h * p.v_h + copy_t * p.v_t + copy_piece * 8;
  auto copy = [&](int i, int stage) {  // chunk i
    const uint16_t *k, *v;
    long long kt, vt;
    int n;
    if (i < chunks1) {
      const long long t0 = (long long)i * KC;
      k = k1 + t0 * p.k_t;
      v = v1 + t0 * p.v_t;
      kt = p.k_t * EACH, vt = p.v_t * EACH;
      n = int(min(n1 - t0, (long long)KC));
    } else {
      const int s = __popc(__ballot_sync(0xffffffffu, upto <= i - chunks1));
      const long long t0 = (long long)(i - chunks1 - __shfl_sync(0xffffffffu, upto - chunks2, s)) * KC;
      const long long len = __shfl_sync(0xffffffffu, len2, s), r = (long long)b * p.R + first + s;
      k = p.k2 + r * p.k2_b + h * p.k2_h + (t0 + copy_t) * p.k2_t + copy_piece * 8;
      v = p.v2 + r * p.v2_b + h * p.v2_h + (t0 + copy_t) * p.v2_t + copy_piece * 8;
      kt = p.k2_t * EACH, vt = p.v2_t * EACH;
      n = int(min(len - t0, (long long)KC));
    }
    const uint32_t at = mem + uint32_t(stage * kChunkBytes);
    // key u * EACH + copy_t: pieces of keys exchanged by 4 in odd ones, of values by the key's last three bits
    const uint32_t k_at = at + uint32_t(copy_t * HD * 2 + ((copy_piece ^ ((copy_t & 1) << 2)) * 16));
    const uint32_t v_at = at + uint32_t(KC * HD * 2 + copy_t * HD * 2), v_piece = uint32_t(copy_piece ^ copy_t) * 16;
    if (n == KC) {
#pragma unroll
      for (int u = 0; u < KC / EACH; ++u, k += kt, v += vt) {
        copy16(k_at + u * EACH * HD * 2, k);
        copy16(v_at + u * EACH * HD * 2 + (v_piece ^ (((u * EACH) & 7) * 16)), v);
      }
    } else {
#pragma unroll
      for (int u = 0; u < KC / EACH; ++u, k += kt, v += vt) {
        const bool there = u * EACH + copy_t < n;
        copy16_or_zero(k_at + u * EACH * HD * 2, there ? k : p.q, there);
        copy16_or_zero(v_at + u * EACH * HD * 2 + (v_piece ^ (((u * EACH) & 7) * 16)), there ? v : p.q, there);
      }
    }
  };
  const int step = int(nsplit) * nw;
  int at = int(rank) * nw + warp;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (at + s * step < total) copy(at + s * step, s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  int stage = 0;
#pragma unroll 1
  for (; at < total; at += step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();  // the other lanes' copies too; and the stage that is filled next has been read
    if (at + (kStages - 1) * step < total) copy(at + (kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    int n, seg = -1;  // keys there; whose: -1 all rows'
    if (at < chunks1) {
      n = int(min(n1 - (long long)at * KC, (long long)KC));
    } else {
      seg = __popc(__ballot_sync(0xffffffffu, upto <= at - chunks1));
      n = int(min(__shfl_sync(0xffffffffu, len2, seg) - (long long)(at - chunks1 - __shfl_sync(0xffffffffu, upto - chunks2, seg)) * KC, (long long)KC));
    }
    const uint32_t keys_at = mem + uint32_t(stage * kChunkBytes), values_at = keys_at + KC * HD * 2;
    float s[MT][NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float odd[MT][4] = {};  // two chains of products
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
#pragma unroll
      for (int ch = 0; ch < HD / 32; ++ch) {
        const uint4 k = tc::ld_shared_v4(keys_at + uint32_t((j * 8 + g) * HD * 2 + (((ch * 4 + c) ^ ((g & 1) << 2)) * 16)));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<BF16>(s[mt][j], qf[mt][2 * ch], k.x, k.y);
          mma16816<BF16>(odd[mt], qf[mt][2 * ch + 1], k.z, k.w);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][j][e] += odd[mt][e];
    }
    uint32_t pr[MT][NT][2];
    const bool some = n < KC || seg >= 0;  // scores that do not count
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (some) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j * 8 + 2 * c + (e & 1) >= n || (seg >= 0 && seg != own[mt][e >> 1])) s[mt][j][e] = -INFINITY;
            else s[mt][j][e] *= p.scale_log2;
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][j][e] *= p.scale_log2;
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[mt][j][e]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
      }
      // The reference exponent of a row moves only when its maximum has grown by more than that.
      constexpr float kGrowth = weight_growth(BF16), kLift = weight_lift(BF16);
      if (__any_sync(0xffffffffu, mx[0] > m[mt][0] + kGrowth || mx[1] > m[mt][1] + kGrowth)) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float now = fmaxf(m[mt][half], mx[half]), corr = now == m[mt][half] ? 1.f : ex2(m[mt][half] - now);
          m[mt][half] = now;
          l[mt][half] *= corr;
#pragma unroll
          for (int j = 0; j < DT; ++j) {
            o[mt][j][2 * half] *= corr;
            o[mt][j][2 * half + 1] *= corr;
          }
        }
      }
      const float base[2] = {m[mt][0] == -INFINITY ? 0.f : m[mt][0] - kLift, m[mt][1] == -INFINITY ? 0.f : m[mt][1] - kLift};  // (no key of this row yet)
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
    // the values of 16 keys and 16 dimensions at a time, turned: two operands of two registers
    uint32_t vr[KC / 16][DT / 2][4];
    bool finite = true;
#pragma unroll
    for (int st = 0; st < KC / 16; ++st)
#pragma unroll
      for (int j = 0; j < DT / 2; ++j) {
        const int t = st * 16 + (lane & 15), piece = 2 * j + (lane >> 4);
        ldmatrix_turned(vr[st][j], values_at + uint32_t(t * HD * 2 + ((piece ^ (t & 7)) * 16)));
      }
    // Own keys are those of some rows only: the others' weights are zero, but a zero times an infinity is not, so then their results stay out.
    if (seg >= 0) {
      uint32_t zero = 0;
#pragma unroll
      for (int st = 0; st < KC / 16; ++st)
#pragma unroll
        for (int j = 0; j < DT / 2; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) zero = times_zero<BF16>(vr[st][j][x], zero);
      finite = __all_sync(0xffffffffu, (zero & 0x7fff7fffu) == 0);
    }
    auto product = [&](auto plain) {
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        float add[MT][4] = {};
#pragma unroll
        for (int st = 0; st < KC / 16; ++st)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint32_t a[4] = {pr[mt][2 * st][0], pr[mt][2 * st][1], pr[mt][2 * st + 1][0], pr[mt][2 * st + 1][1]};
            mma16816<BF16>(plain.value ? o[mt][j] : add[mt], a, vr[st][j / 2][(j & 1) * 2], vr[st][j / 2][(j & 1) * 2 + 1]);
          }
        if (!plain.value) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (seg == own[mt][e >> 1]) o[mt][j][e] += add[mt][e];
        }
      }
    };
    if (finite) product(std::true_type{});
    else product(std::false_type{});
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();  // the chunks' memory is the part's now
  // the warps' parts, the block's, the cluster's
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 1);
      l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 2);
      const int r = mt * 16 + half * 8 + g;
      if (r >= rows) continue;
      float* d = part + warp * kPart + r * PITCH;
#pragma unroll
      for (int j = 0; j < DT; ++j) *reinterpret_cast<float2*>(d + j * 8 + 2 * c) = make_float2(o[mt][j][2 * half], o[mt][j][2 * half + 1]);
      if (c == 0) {
        d[HD] = m[mt][half];
        d[HD + 1] = l[mt][half];
      }
    }
  __syncthreads();
  // a warp a row: its maximum and sum over the warps, and their weights (a sum of NaN stays one)
  for (int r = warp; r < rows; r += nw) {
    float mw = -INFINITY, lw = 0.f, mx;
    if (lane < nw) {
      mw = part[lane * kPart + r * PITCH + HD];
      lw = part[lane * kPart + r * PITCH + HD + 1];
    }
    mx = mw;
#pragma unroll
    for (int o = kRowsWarps / 2; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float ww = lw == 0.f ? 0.f : ex2(mw - mx);
    float sum = ww * lw;
#pragma unroll
    for (int o = kRowsWarps / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < nw) part[lane * kPart + r * PITCH + HD + 1] = ww;
    if (lane == 0) {
      total_of[2 * r] = mx;
      total_of[2 * r + 1] = sum;
    }
  }
  if (nsplit > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  __syncthreads();
  const int Hq = p.Hkv * p.G;
  auto put4 = [&](int r, int e, float4 v, float mx, float sum) {  // elements e .. e + 3 of the tile's row r
    const int rr = row0 + r;
    if (p.parts) {
      const size_t at = ((size_t(bh) * ((p.R * p.G + kTcRows - 1) / kTcRows) + rr / kTcRows) * p.n_parts + p.n_parts - 1) * p.part_rows + rr % kTcRows;
      *reinterpret_cast<float4*>(p.parts + at * HD + e) = v;
      if (e == 0) *reinterpret_cast<float2*>(p.stats + at * 2) = make_float2(mx, sum);
      return;
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    *reinterpret_cast<uint2*>(p.out + ((size_t(b) * p.R + rr / p.G) * Hq + h * p.G + rr % p.G) * HD + e) =
        make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
  };
  // Four elements a thread.  In a cluster a block finishes every nsplit-th of them: the others send it theirs.
  constexpr int Q4 = HD / 4;
  for (int i = threadIdx.x; i < rows * Q4; i += blockDim.x) {
    const int r = i / Q4, e = (i % Q4) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, const float4& v) {
      acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
    };
#pragma unroll 4
    for (int w = 0; w < nw; ++w) add(part[w * kPart + r * PITCH + HD + 1], *reinterpret_cast<const float4*>(part + w * kPart + r * PITCH + e));
    if (nsplit == 1) {
      put4(r, e, acc, total_of[2 * r], total_of[2 * r + 1]);
    } else {
      const uint32_t to = tc::mapa(tc::smem_u32(gathered + (rank * (ROWS * Q4 / nsplit) + i / nsplit) * 4), uint32_t(i) % nsplit);
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(acc.x), "f"(acc.y), "f"(acc.z), "f"(acc.w) : "memory");
    }
  }
  // (who waits for this kernel waits for the one before it too)
  if (p.parts) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nsplit == 1) return;
  for (int i = threadIdx.x; i < rows * int(nsplit); i += blockDim.x) {
    const int r = i / int(nsplit);
    const uint32_t to = tc::mapa(tc::smem_u32(stats + (rank * ROWS + r) * 2), uint32_t(i) % nsplit);
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(total_of[2 * r]), "f"(total_of[2 * r + 1]) : "memory");
  }
  tc::cluster_sync();  // everything has arrived, and nobody reads another's any more
  for (int i = int(rank) + threadIdx.x * int(nsplit); i < rows * Q4; i += int(blockDim.x) * int(nsplit)) {
    const int r = i / Q4, e = (i % Q4) * 4;
    float mx = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (uint32_t x = 0; x < nsplit; ++x) mx = fmaxf(mx, stats[(x * ROWS + r) * 2]);
#pragma unroll 4
    for (uint32_t x = 0; x < nsplit; ++x) {
      const float2 ml = *reinterpret_cast<const float2*>(stats + (x * ROWS + r) * 2);
      const float4 v = *reinterpret_cast<const float4*>(gathered + (x * (ROWS * Q4 / nsplit) + i / nsplit) * 4);
      const float w = ml.y == 0.f ? 0.f : ex2(ml.x - mx);
      sum = fmaf(w, ml.y, sum);
      acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
    }
    put4(r, e, acc, mx, sum);
  }
}

template <int HD, int MT>
size_t rows_smem(int warps) {
  constexpr int ROWS = 16 * MT;
  return size_t(warps) * kStages * kChunkBytes + (ROWS * HD + 2 * kMaxSplit * ROWS + 2 * ROWS) * 4;
}

// Blocks of `warps` warps, in clusters of `split`, that the device holds at once; 0: it holds no such cluster
template <int HD, int MT, bool BF16>
int64_t resident_blocks(int split, int warps, int sm_count) {
  static std::atomic<int> known[kMaxSplit + 1][kRowsWarps + 1];  // one more than that; one kind of device: asked once per process
  std::atomic<int>& k = known[split][warps];
  const int before = k.load(std::memory_order_relaxed);
  if (before) return before - 1;
  auto kern = rows_attn_kernel<HD, MT, BF16>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(split));
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = rows_smem<HD, MT>(warps);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int held = 0;
  if (cudaOccupancyMaxActiveClusters(&held, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    held = -1;
  }
  const int64_t n = slots_held(held, split, sm_count);
  k.store(int(n) + 1, std::memory_order_relaxed);
  return n;
}

template <int HD, int MT, bool BF16>
RowsChoice choose_for(int64_t B, int64_t R, int G, int n_kv_heads, int64_t keys, int64_t keys2, int sm_count) {
  constexpr int ROWS = 16 * MT, KC = HD == 64 ? 32 : 16;
  const int64_t items = B * n_kv_heads * ((R * G + ROWS - 1) / ROWS);
  const int64_t chunks = std::min<int64_t>((keys + KC - 1) / KC + std::min<int64_t>((ROWS - 1) / G + 1, R) * ((keys2 + KC - 1) / KC), 1 << 30);
  return choose_rows(uint32_t(items), uint32_t(chunks), [&](int split, int warps) { return resident_blocks<HD, MT, BF16>(split, warps, sm_count); });
}

template <int HD, int MT, bool BF16>
int allow_rows() {  // what the occupancy query and the launch need set
  auto kern = rows_attn_kernel<HD, MT, BF16>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), rows_smem<HD, MT>(kRowsWarps));
  if (rc) return rc;
  ASRQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  return ASRQ_OK;
}

template <int HD, int MT, bool BF16>
int launch_rows(RowsParams p, int64_t B, int sm_count, cudaStream_t stream) {
  constexpr int ROWS = 16 * MT;
  p.tiles = (p.R * p.G + ROWS - 1) / ROWS;
  const int64_t items = B * p.Hkv * p.tiles;
  auto kern = rows_attn_kernel<HD, MT, BF16>;
  const RowsChoice choice = choose_for<HD, MT, BF16>(B, p.R, p.G, p.Hkv, p.keys, p.k2 ? p.keys2 : 0, sm_count);
  const int split = choice.split, warps = choice.warps;
  const size_t smem = rows_smem<HD, MT>(warps);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(items * split));
  cfg.blockDim = dim3(32 * warps);
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

// The row kernel's time in us, by its units above: 1.2 each, more with many dimensions or rows to a warp (measured: 1.1 to 1.5, 1.2 to 1.5, 1.6 to 1.75).
double rows_estimate(int64_t B, int64_t R, int G, int n_kv_heads, int hd, int64_t keys, int64_t keys2, int sm_count) {
  if (hd == 128) return 1.3 * double(choose_for<128, 1, false>(B, R, G, n_kv_heads, keys, keys2, sm_count).cost);
  if (R * G > 16) return 1.65 * double(choose_for<64, 2, false>(B, R, G, n_kv_heads, keys, keys2, sm_count).cost);
  return 1.2 * double(choose_for<64, 1, false>(B, R, G, n_kv_heads, keys, keys2, sm_count).cost);
}

// Whether the tensor-core kernel takes a call, and how it divides it.  Its blocks walk tiles of keys at about 1.15 us each (1.3 where own keys follow),
// one more for a unit of work and two for the start, however few of the 128 rows there are; items that fill the chip are left whole, the rest
// divided so that it is filled once more, and a join is worth about 4, of up to 64 rows of 128 dimensions 3.  us, the row kernel first: heads of 64 on 1500 keys, 16 utterances of 5 rows
// 23 | 29, 20 rows 44 | 29, 64 rows 74 | 30; 4 of 32 rows 14 | 17, 64 rows 22 | 18; 1 of 64 rows 11 | 10; on 150 keys, 16 of 20 rows 10.7 | 8.7, of 5 5.4 | 8.7;
// heads of 128 on 6000 keys, 16 utterances of 8 rows 64 | 74, 20 rows 107 | 76, 64 rows 279 | 84; behind 6000 shared keys 200 own ones, 4 utterances of 16
// beams 34 | 41, 32 beams 56 | 51.
TcPlan tc_plan(int64_t B, int64_t R, int G, int n_kv_heads, int hd, int64_t keys, int64_t keys2, int sm_count) {
  const int64_t rows = R * G, tiles = (rows + kTcRows - 1) / kTcRows, items = B * n_kv_heads * tiles, step = hd == 64 ? 96 : 64;
  const int64_t key_tiles = (keys + step - 1) / step, slots = 2 * sm_count;
  const bool own = keys2 > 0;
  const int forced = option(kOptRowsKernel);
  if (keys == 0 || kTcRows % G != 0 || forced == 1 || (forced != 2 && (rows <= 16 || keys < 64))) return {0, 0};
  const int64_t whole = own ? 0 : items / slots * slots, rest = items - whole, first = whole / slots * (key_tiles + 1);
  TcPlan plan = {own ? 0 : items, own ? 0 : 1};
  int64_t least = rest == 0 ? 0 : own ? INT64_MAX : key_tiles + 1;
  for (int s = own ? 1 : 2; s <= kMaxParts && rest > 0 && (s == 1 || key_tiles >= 2 * s); ++s) {
    const int64_t cost = (rest * s + slots - 1) / slots * ((key_tiles + s - 1) / s + 1) + (hd == 128 && rows <= 64 ? 3 : 4) + s / 8;
    if (cost < least) {
      least = cost;
      plan = {whole, s};
    }
  }
  if (forced == 2) return plan;
  double us = (own ? 1.3 : 1.15) * double(first + least + 2);
  if (own) us += rows_estimate(B, R, G, n_kv_heads, hd, 0, keys2, sm_count);
  return us < rows_estimate(B, R, G, n_kv_heads, hd, keys, keys2, sm_count) ? plan : TcPlan{0, 0};
}
int allow_all() {
  static std::atomic<uint64_t> devices;  // that have it
  int dev = 0;
  ASRQ_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (devices.load(std::memory_order_relaxed) & bit) return ASRQ_OK;
  int rc = allow_rows<64, 1, false>();
  if (!rc) rc = allow_rows<64, 1, true>();
  if (!rc) rc = allow_rows<64, 2, false>();
  if (!rc) rc = allow_rows<64, 2, true>();
  if (!rc) rc = allow_rows<128, 1, false>();
  if (!rc) rc = allow_rows<128, 1, true>();
  if (!rc) devices.fetch_or(bit, std::memory_order_relaxed);
  return rc;
}
size_t part_count(int64_t B, int64_t R, int G, int n_kv_heads, const TcPlan& plan, bool own) {  // rows of all parts
  if (plan.split == 0) return 0;
  const int64_t items = B * n_kv_heads * ((R * G + kTcRows - 1) / kTcRows);
  return size_t(items - plan.whole) * (plan.split + own) * part_rows_of(R * G);
}

size_t rows_attention_scratch_bytes(int64_t B, int64_t R, int n_q_heads, int n_kv_heads, int hd, int64_t keys, int64_t keys2, int sm_count) {
  const int G = n_q_heads / n_kv_heads;
  return allow_all() ? 0 : part_count(B, R, G, n_kv_heads, tc_plan(B, R, G, n_kv_heads, hd, keys, keys2, sm_count), keys2 > 0) * (hd + 2) * sizeof(float);
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
  TcPlan plan = {0, 0};
  auto launch = [&](const RowsParams& x) {
    if (hd == 128) return bf16 ? launch_rows<128, 1, true>(x, B, sm_count, stream) : launch_rows<128, 1, false>(x, B, sm_count, stream);
    if (R * x.G > 16) return bf16 ? launch_rows<64, 2, true>(x, B, sm_count, stream) : launch_rows<64, 2, false>(x, B, sm_count, stream);
    return bf16 ? launch_rows<64, 1, true>(x, B, sm_count, stream) : launch_rows<64, 1, false>(x, B, sm_count, stream);
  };
  int rc = allow_all();
  if (rc) return rc;
  // (the tensor-core kernel's copies know no two elements at one place but along whole dimensions of keys, and it hides scores before it scales them)
  auto apart = [](int64_t n, int64_t stride) { return n == 1 || stride != 0; };
  if (status && p.scale_log2 > 0.f && apart(keys, ks[2]) && apart(keys, vs[2]) && apart(B, qs[0]) && apart(R, qs[1]) && apart(n_q_heads, qs[2]))
    plan = tc_plan(B, R, p.G, n_kv_heads, hd, keys, k2 ? keys2 : 0, sm_count);
  if (plan.split > 0) {
    const size_t rows = part_count(B, R, p.G, n_kv_heads, plan, k2 != nullptr), need = rows * (hd + 2) * sizeof(float);
    const bool kept = need == 0 || (scratch && scratch_bytes >= need);
    if (!kept && !k2) plan = {B * n_kv_heads * ((R * p.G + kTcRows - 1) / kTcRows), 1};
    if (kept || !k2) {
      float *parts = need && kept ? static_cast<float*>(scratch) : nullptr, *stats = parts ? parts + rows * hd : nullptr;
      rc = rows_attention_tc(p, hd, bf16, B, plan, parts, stats, k2 ? 1 : 0, status, sm_count, stream);
      if (!rc && k2) {
        RowsParams own = p;
        own.keys = 0;
        own.parts = parts, own.stats = stats;
        own.n_parts = plan.split + 1;
        own.part_rows = part_rows_of(R * p.G);
        rc = launch(own);
      }
      return rc ? rc : rows_attention_join(p, hd, bf16, B, plan.whole, parts, stats, plan.split + (k2 ? 1 : 0), stream);
    }
  }
  return launch(p);
}

}  // namespace asrq
