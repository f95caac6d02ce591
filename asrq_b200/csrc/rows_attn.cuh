// What the two kernels of attention over shared keys (rows_attn.cu, rows_attn_tc.cu) have in common.
#pragma once

#include "tcgen05.cuh"

namespace asrq {

struct RowsParams {
  const uint16_t* q;             // row r of utterance b, head h: q + b * q_b + r * q_r + h * q_h
  uint16_t* out;                 // B x R x (Hkv * G) x HD
  const uint16_t *k, *v;         // shared: key t of utterance b, head h at k + b * k_b + h * k_h + t * k_t
  const uint16_t *k2, *v2;       // own: of row b * R + r
  const long long *len, *len2;   // B, or NULL for `keys`; one, or B * R
  long long q_b, q_r, q_h, k_b, k_h, k_t, v_b, v_h, v_t, k2_b, k2_h, k2_t, v2_b, v2_h, v2_t;
  long long keys, keys2;         // room
  int len2_many, R, G, Hkv, tiles;
  float scale_log2;              // scale * log2 e
  // Where the shared keys are the tensor-core kernel's, a row kernel leaves its rows' own keys as one more part: for every utterance, key head and tile of
  // 128 rows n_parts parts of part_rows results of HD values, the row kernel's the last, and in stats as many pairs of maximum (as an exponent of two) and sum.
  float *parts, *stats;
  int n_parts, part_rows;
};
// Both kernels take a row's weights as 2^(s - m + lift), s the scores in units of log 2 and m a maximum that follows s only when s has
// grown by more than `growth`; the parts' sums and values carry the same 2^lift.  bf16 has the exponents of fp32 and needs no lift.  An fp16
// weight lies in 2^(growth + lift) = 2^15 at most, all its bits above 2^-14: lifted by 11, weights keep them down to 2^-25 of the largest and count down to 2^-36 of
// it, so that even 2^24 keys below that would not show in the result.  (Without a lift, weights below 2^-25 of the largest were lost, 40 000 keys of 2^-25 and their
// thousandth of the result with them.)
__host__ __device__ constexpr float weight_growth(bool bf16) { return bf16 ? 8.f : 4.f; }
__host__ __device__ constexpr float weight_lift(bool bf16) { return bf16 ? 0.f : 11.f; }

constexpr int kTcRows = 128, kMaxParts = 64;  // rows of its tile; parts it divides an item's keys into at most
// Rows of a tile's parts: 128, or as many as there are, an odd number: a join reads a row of all parts at once, and at distances of 64 KB they were slower to come
// (64 samples behind 45 000 keys: 57.7 us for 56.3 with 128 rows for 129).
__host__ __device__ constexpr int part_rows_of(int64_t rows) { return int(rows < kTcRows ? rows : kTcRows) | 1; }

// How the tensor-core kernel divides a call's items (utterance, key head, 128 rows): the first `whole` have a block each, the keys of the others
// are divided among `split`, each of which leaves a part.  split 0: the call is not for it.
struct TcPlan {
  int64_t whole;
  int split;
};

// The shared keys of p by tcgen05; room is left behind every item's parts for `more` of them.
int rows_attention_tc(const RowsParams& p, int hd, bool bf16, int64_t B, const TcPlan& plan, float* parts, float* stats, int more, void* status, int sm_count,
                      cudaStream_t stream);

// The results of the items from `whole` on, from n_parts parts each.
int rows_attention_join(const RowsParams& p, int hd, bool bf16, int64_t B, int64_t whole, const float* parts, const float* stats, int n_parts, cudaStream_t stream);

}  // namespace asrq
