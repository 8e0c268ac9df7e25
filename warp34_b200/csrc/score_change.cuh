// What warp34_paged_attention_scored_* changes between the product of a query with a key and the softmax, shared by the attention kernels:
//
//   t = sm_scale q k;   t <- cap tanh(t / cap);   t <- t - slope[head] |position of the query - position of the key|
//   key visible iff  first(token) <= position <= last(token)
//
// Kernels hold scores in units of log2(e) (weights are powers of two), so the factors here are as well.
// tanh(x) = 1 - 2 / (e^(2 x) + 1), two special-function instructions, off by less than 5 x 2^-23 of the cap: in units of 2^-23, with
// u = e^(2 x), the power (2^-22 of itself, and 2^-23 |2 x| from its exponent's rounding) 2 u / (u + 1)^2 (2 + |2 x|), the sum's rounding and the
// reciprocal 3 / (u + 1), the cap in log2(e) units and the last rounding 1.5 |tanh x|; together 4.8 at most, at 2 x about -3.  That is 6e-4
// of a weight at the largest cap that is accepted and 3e-5 at a cap of 50.  (tanh.approx, one instruction, is off by 2^-11 of the cap: 2.5 % of a weight at a cap of 50.)
// A penalty is taken off in fp32 (its slope in log2(e) units 2 x 2^-24, the score's rounding 2^-24): a weight is off by 3 x 2^-24 of the largest
// penalty among the keys that count.
// Included by tq4_attention.cu.
#pragma once

namespace w34 {

constexpr float kMaxSoftcap = 1024.0f, kMinSoftcap = 1.0f / 1024.0f;

struct ScoreChange {
    float cap = 0.0f;         // x log2(e); 0: scores are not capped
    float cap_arg = 0.0f;     // 2 / cap: what makes a score the exponent of e^(2 t / cap)
    const float* slopes = nullptr;           // [q heads]
    const int32_t* key_begin = nullptr;      // [tokens] first key, or null
    const int32_t* key_end = nullptr;        // [tokens] key behind the last, in place of causality, or null
};

// First and last key of a row.  SCORED: the token's own limits as well.
template <bool SCORED>
__device__ __forceinline__ int row_first_key(const warp34_attention_batch& b, const ScoreChange& sc, const ReqGeom& g, int q_off) {
    int m = row_min_kv(b, g, q_off);
    if (SCORED && sc.key_begin != nullptr) m = max(m, sc.key_begin[g.q_start + q_off]);
    return m;
}
template <bool SCORED>
__device__ __forceinline__ int row_last_key(const warp34_attention_batch& b, const ScoreChange& sc, const ReqGeom& g, int q_off) {
    if (SCORED && sc.key_end != nullptr) return min(max(sc.key_end[g.q_start + q_off], 0), g.seq_after) - 1;
    return row_max_kv(b, g, q_off);
}

// A score's cap.
__device__ __forceinline__ float capped_score(const ScoreChange& sc, float t) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t * sc.cap_arg));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
    return __fmaf_rn(-2.0f * sc.cap, r, sc.cap);
}
// The change of one score: `slope` in log2(e) units, `away` position of the query less that of the key as a float (from one conversion for a
// row and a block of keys: int to float is as dear as a reciprocal).  Without a branch, for the stream kernels: a cap is computed and selected
// in any case, so that the products of the next page and the rest of a step's work fill its latency (64 sequences of 8192 to 32768, capped: 598
// us with a branch around it, 537 without).
__device__ __forceinline__ float changed_score(const ScoreChange& sc, float t, float slope, float away) {
    const float capped = capped_score(sc, t);
    asm("{\n\t.reg .pred p;\n\tsetp.neu.f32 p, %3, 0f00000000;\n\tselp.f32 %0, %1, %2, p;\n\t}" : "=f"(t) : "f"(capped), "f"(t), "f"(sc.cap));
    return __fmaf_rn(-slope, fabsf(away), t);
}
__device__ __forceinline__ float max_of(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 32 products of one row, times `factor`, as changed scores, for the chunk kernel; `away` position of the query less that of the first key.
// Two scores at a time, and branches outside the loops.  (A branch for every score keeps the chains of power, sum and reciprocal
// from running side by side: 8 x 2048 BF16 tokens after 8192 3.8 instead of 3.3 ms.)
__device__ __forceinline__ void change_scores(const ScoreChange& sc, float (&t)[32], float factor, float slope, float away) {
    if (sc.cap != 0.0f) {
        const Two k = two_of(factor * sc.cap_arg, factor * sc.cap_arg), one = two_of(1.0f, 1.0f), cap = two_of(sc.cap, sc.cap),
                  cap2 = two_of(-2.0f * sc.cap, -2.0f * sc.cap);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const Two x = mul_two(two_of(t[i], t[i + 1]), k);
            float e0, e1, r0, r1;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(first_of(x)));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(second_of(x)));
            const Two e = add_two(two_of(e0, e1), one);
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(first_of(e)));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(second_of(e)));
            const Two y = fma_two(two_of(r0, r1), cap2, cap);
            t[i] = first_of(y);
            t[i + 1] = second_of(y);
        }
    } else {
        const Two f = two_of(factor, factor);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const Two y = mul_two(two_of(t[i], t[i + 1]), f);
            t[i] = first_of(y);
            t[i + 1] = second_of(y);
        }
    }
    if (sc.slopes != nullptr) {
#pragma unroll
        for (int i = 0; i < 32; ++i) t[i] = __fmaf_rn(-slope, fabsf(away - (float)i), t[i]);
    }
}
__device__ __forceinline__ float row_slope(const ScoreChange& sc, int q_head) { return sc.slopes != nullptr ? sc.slopes[q_head] * 1.4426950408889634f : 0.0f; }

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

}  // namespace w34
