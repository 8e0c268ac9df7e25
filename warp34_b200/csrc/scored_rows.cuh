// Attention with changed scores, a row at a time in fp32, over every layer format and any strides: the kernel for calls that the
// tensor-core kernels do not take (no workspace, other packings, mixed 8-bit formats, WARP34_B200_EXEC_FLAG_PRECISE_ATTENTION), and the
// second look at rows that came out non-finite.  The latter because a product of a tile's weights with its V rows meets every row of
// the tile with every key of it: a NaN or infinity in the V of a key that one row must not see (another document's, say) is 0 x NaN there.
// A row that sees every such key itself is what it must be, and is left alone (scored_bad_rows: one look at the keys of its tile, bound by
// memory.  Computing such rows again, key by key: 74 ms instead of 0.67 for 2048 BF16 tokens after 2048, 24 / 4 heads, behind one NaN in the
// prefix; 0.32 without it).
// Included by tq4_attention.cu.
#pragma once

namespace w34 {

// A stored row's columns [8 lane, + 8) as they lie in memory (TQ4: in the rotated basis), so that several rows are on their way before the
// first is used.
struct ScoredRaw { uint32_t w[4]; float d; };
__device__ __forceinline__ void scored_load(ScoredRaw& r, const uint8_t* row, int format, int lane, int aligned) {
    if (format == WARP34_KV_FORMAT_TQ4) {
        const uint8_t* half = row + kTq4BlockBytes * (lane >> 4);
        const uint16_t* codes = reinterpret_cast<const uint16_t*>(half + 2 + 4 * (lane & 15));
        r.w[0] = codes[0];
        r.w[1] = codes[1];
        r.w[2] = *reinterpret_cast<const uint16_t*>(half);
    } else if (format == WARP34_KV_FORMAT_BF16) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(row) + 8 * lane;
        if (aligned) {
            const uint4 q = *reinterpret_cast<const uint4*>(src);
            r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r.w[i] = (uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16);
        }
    } else {
        const bool fp8 = format == WARP34_KV_FORMAT_FP8_E4M3;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(row + (fp8 ? 8 * lane : 68 * (lane >> 3) + 4 + 8 * (lane & 7)));
        r.w[0] = codes[0];
        r.w[1] = codes[1];
        r.d = *reinterpret_cast<const float*>(row + (fp8 ? kHeadDim + 4 * (lane >> 4) : 68 * (lane >> 3)));
    }
}
// `centroid`: of a code; every lane of the warp comes here.
template <class Centroid>
__device__ __forceinline__ void scored_values(const ScoredRaw& r, int format, Centroid centroid, float (&x)[8]) {
    if (format == WARP34_KV_FORMAT_TQ4) {
        const float d = __half2float(__ushort_as_half((unsigned short)r.w[2]));
        const uint32_t w = r.w[0] | (r.w[1] << 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = d * centroid((w >> (4 * i)) & 15u);
    } else if (format == WARP34_KV_FORMAT_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(r.w[i] << 16);
            x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t a, b;
            if (format == WARP34_KV_FORMAT_FP8_E4M3) kv8x4_to_f16x4<WARP34_KV_FORMAT_FP8_E4M3>(r.w[i], a, b);
            else kv8x4_to_f16x4<WARP34_KV_FORMAT_Q8_0>(r.w[i], a, b);
            const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a)), fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
            x[4 * i] = r.d * fa.x; x[4 * i + 1] = r.d * fa.y; x[4 * i + 2] = r.d * fb.x; x[4 * i + 3] = r.d * fb.y;
        }
    }
}

// Sums over the lanes of N values a lane (a power of two): lane l ends with the sum of value l N / 32.
template <int N>
__device__ __forceinline__ float scored_sums(float (&v)[N], int lane) {
    int step = 16;
#pragma unroll
    for (int n = N; n > 1; n >>= 1) {
        const bool upper = (lane & step) != 0;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float keep = upper ? v[i + n / 2] : v[i], give = upper ? v[i] : v[i + n / 2];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, step);
        }
        step >>= 1;
    }
    float s = v[0];
#pragma unroll
    for (int d = 16 / N; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    return s;
}

struct ScoredRow {
    const warp34_kv_layer_layout* layout;
    const warp34_attention_batch* batch;
    const ScoreChange* sc;
    const void* q_in;
    int io_bf16, num_q_heads, gqa;
};

// Every `step`th group of KEYS keys, from the `first` on, of [lo, hi] of one query row by one warp: columns [8 lane, + 8) of sum w V (stored
// basis), running maximum (log2 units) and mass.  The keys' rows are on their way at once and their products summed over the lanes
// together, a key's score to 32 / KEYS lanes (keys one after the other: 1 us a key, on TQ4 with its table in constant memory 4).
// Four keys where registers allow (0.4 us a key and warp with 14 warps an SM), two in the merge kernel, whose registers bound its blocks an SM, one
// where it stands inside the chunk kernel (with four there, 8 x 2048 TQ4 tokens after 8192 took 0.6 % longer without coming here).
template <int KEYS>
__device__ __forceinline__ void scored_row_keys(const ScoredRow& p, int req, int q_off, int q_head, int lo, int hi, int first, int step, float (&acc)[8],
                                             float& m, float& l) {
    const int lane = threadIdx.x & 31, kv_head = q_head / p.gqa;
    const warp34_attention_batch& b = *p.batch;
    const warp34_kv_layer_layout& lay = *p.layout;
    const ReqGeom g = load_req(b, req);
    const int32_t* blocks = b.block_tables + (size_t)req * b.max_blocks_per_req;
    const uint8_t* k_head = (const uint8_t*)(uintptr_t)lay.k_base + (size_t)kv_head * lay.k_head_stride_bytes;
    const uint8_t* v_head = (const uint8_t*)(uintptr_t)lay.v_base + (size_t)kv_head * lay.v_head_stride_bytes;
    const int aligned = ((lay.k_base | lay.v_base | lay.k_page_stride_bytes | lay.k_head_stride_bytes | lay.k_token_stride_bytes | lay.v_page_stride_bytes |
                          lay.v_head_stride_bytes | lay.v_token_stride_bytes) & 15u) == 0u;
    lo = max(lo, row_first_key<true>(b, *p.sc, g, q_off));
    hi = min(hi, row_last_key<true>(b, *p.sc, g, q_off));
    float q[8];
    load8(p.q_in, ((size_t)(g.q_start + q_off) * p.num_q_heads + q_head) * kHeadDim, lane, p.io_bf16, q);
    float scale = b.sm_scale * 1.4426950408889634f;
    if (lay.k_format == WARP34_KV_FORMAT_TQ4) {
        sign8(q, lane);
        butterfly8<5>(q, lane);
        scale *= 0.0625f;
    }
    const float slope = row_slope(*p.sc, q_head), mine = tq4_centroid(lane & 15);
    const auto centroid = [&](uint32_t code) { return __shfl_sync(0xffffffffu, mine, (int)code); };
    const int q_pos = g.ctx_before + q_off;
    m = -1e30f;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
    if (lo > hi) return;
    const int last = hi / KEYS;
    auto page_of = [&](int n) { return n <= last ? block_table_page(blocks, n / (kPageTokens / KEYS), b.max_blocks_per_req, kInScalar) : 0; };
    int n = lo / KEYS + first, page = page_of(n);
#pragma unroll 1
    for (; n <= last; n += step) {
        ScoredRaw raw[KEYS];      // K, then V
        const auto load = [&](const uint8_t* run, size_t token_stride, int format) {
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {      // (keys outside the row's are not looked at)
                scored_load(raw[i], run + (size_t)(min(max(KEYS * n + i, lo), hi) & 15) * token_stride, format, lane, aligned);
            }
        };
        load(k_head + (size_t)page * lay.k_page_stride_bytes, lay.k_token_stride_bytes, lay.k_format);
        float s[KEYS], x[8];
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            scored_values(raw[i], lay.k_format, centroid, x);
            s[i] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i] = __fmaf_rn(q[e], x[e], s[i]);
        }
        load(v_head + (size_t)page * lay.v_page_stride_bytes, lay.v_token_stride_bytes, lay.v_format);
        page = page_of(n + step);
        const int pos = KEYS * n + lane / (32 / KEYS);      // the key whose score ends in this lane
        const bool seen = pos >= lo && pos <= hi;
        float t = scored_sums(s, lane) * scale;
        if (p.sc->cap != 0.0f) t = capped_score(*p.sc, t);
        t = __fmaf_rn(-slope, (float)abs(q_pos - pos), t);
        float top = seen ? t : -1e30f;
#pragma unroll
        for (int d = 32 / KEYS; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float m_new = fmaxf(m, top), alpha = ex2(m - m_new), w = seen ? ex2(t - m_new) : 0.0f;
        float sum = w;
#pragma unroll
        for (int d = 32 / KEYS; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        m = m_new;
        l = l * alpha + sum;
        if (l != l) return;      // a NaN in the query or in a key: the row is NaN whatever follows
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= alpha;
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            if (KEYS * n + i < lo || KEYS * n + i > hi) continue;
            const float wi = __shfl_sync(0xffffffffu, w, 32 / KEYS * i);
            scored_values(raw[i], lay.v_format, centroid, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = __fmaf_rn(wi, x[e], acc[e]);
        }
    }
}

// Keys whose rows reach every row that sees them: K rows with a NaN, V rows with a NaN or infinity.  First and last position (none: first > last).
struct ScoredBad {
    int k_first = 0x7fffffff, k_last = -1, v_first = 0x7fffffff, v_last = -1;
    // Whether a row that sees keys [lo, hi], of a tile whose keys this is about, is non-finite of its own: it sees such a key, and no V row it
    // does not see can have reached it.  (Where neither holds, an operand has left the range of the tensor cores' type.)
    __device__ __forceinline__ bool explains(int lo, int hi) const {
        const bool v = v_first <= v_last;
        if (v && (v_first < lo || v_last > hi)) return false;
        return (v && lo <= hi) || (k_first >= lo && k_first <= hi) || (k_last >= lo && k_last <= hi);
    }
};

// The 16 rows of a (page, head) in canonical packing: the lane's part of a bit for each that holds a NaN or, with INFINITIES, an infinity.  A
// lane looks at scales (TQ4, Q8_0), at scales and eight codes of every row (FP8), or at 16 bytes of every row (BF16).
template <bool INFINITIES>
__device__ __forceinline__ uint32_t scored_bad_scales(const uint8_t* run, size_t token_stride, int format, int lane) {
    constexpr uint32_t f16 = INFINITIES ? 0x7bffu : 0x7c00u, f32 = INFINITIES ? 0x7f7fffffu : 0x7f800000u;
    if (format == WARP34_KV_FORMAT_TQ4) {
        const uint32_t d = *reinterpret_cast<const uint16_t*>(run + (size_t)(lane >> 1) * token_stride + kTq4BlockBytes * (lane & 1));
        return ((d & 0x7fffu) > f16 ? 1u : 0u) << (lane >> 1);
    }
    if (format == WARP34_KV_FORMAT_FP8_E4M3) {
        const uint32_t d = *reinterpret_cast<const uint32_t*>(run + (size_t)(lane >> 1) * token_stride + kHeadDim + 4 * (lane & 1));
        return ((d & 0x7fffffffu) > f32 ? 1u : 0u) << (lane >> 1);
    }
    uint32_t bad = 0u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = (lane >> 2) + 8 * i;
        const uint32_t d = *reinterpret_cast<const uint32_t*>(run + (size_t)t * token_stride + 68 * (lane & 3));
        bad |= ((d & 0x7fffffffu) > f32 ? 1u : 0u) << t;
    }
    return bad;
}
template <bool INFINITIES>
__device__ __forceinline__ uint32_t scored_bad_elements(const uint8_t* run, size_t token_stride, int format, int lane) {
    constexpr uint32_t b16 = INFINITIES ? 0x7f7fu : 0x7f80u;
    uint32_t bad = 0u;
    if (format == WARP34_KV_FORMAT_BF16) {
#pragma unroll 2
        for (int t = 0; t < 16; ++t) {
            const uint4 w = *reinterpret_cast<const uint4*>(run + (size_t)t * token_stride + 16 * lane);
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) any = any || (x[i] & 0x7fffu) > b16 || ((x[i] >> 16) & 0x7fffu) > b16;
            bad |= (any ? 1u : 0u) << t;
        }
        return bad;
    }
#pragma unroll 4
    for (int t = 0; t < 16; ++t) {      // the code 0x7f, of either sign, is NaN
        const uint2 w = *reinterpret_cast<const uint2*>(run + (size_t)t * token_stride + 8 * lane);
        const uint32_t any = (((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u;
        bad |= (any != 0u ? 1u : 0u) << t;
    }
    return bad | scored_bad_scales<INFINITIES>(run, token_stride, format, lane);
}

// The keys [lo, hi] of one kv head, every `step`th page from the `first` on, by one warp.  K and V have one format.
__device__ __forceinline__ ScoredBad scored_bad_rows(const ScoredRow& p, int req, int kv_head, int lo, int hi, int first, int step) {
    const int lane = threadIdx.x & 31;
    const warp34_attention_batch& b = *p.batch;
    const warp34_kv_layer_layout& lay = *p.layout;
    const int32_t* blocks = b.block_tables + (size_t)req * b.max_blocks_per_req;
    const uint8_t* k_head = (const uint8_t*)(uintptr_t)lay.k_base + (size_t)kv_head * lay.k_head_stride_bytes;
    const uint8_t* v_head = (const uint8_t*)(uintptr_t)lay.v_base + (size_t)kv_head * lay.v_head_stride_bytes;
    const int format = lay.k_format;
    ScoredBad res;
    if (lo > hi) return res;
    const int last = hi >> 4;
    auto take = [&](int pg, uint32_t k, uint32_t v) {
        const int pos = pg << 4;
        const uint32_t in = (0xffffu << max(lo - pos, 0)) & (0xffffu >> max(pos + 15 - hi, 0));
        k = __reduce_or_sync(0xffffffffu, k) & in;
        v = __reduce_or_sync(0xffffffffu, v) & in;
        if (k != 0u) {
            res.k_first = min(res.k_first, pos + __ffs((int)k) - 1);
            res.k_last = max(res.k_last, pos + 31 - __clz((int)k));
        }
        if (v != 0u) {
            res.v_first = min(res.v_first, pos + __ffs((int)v) - 1);
            res.v_last = max(res.v_last, pos + 31 - __clz((int)v));
        }
    };
    for (int pg0 = (lo >> 4) + first; pg0 <= last; pg0 += 32 * step) {
        const int mine = pg0 + lane * step;      // a lane per page of the table
        const int32_t ids = mine <= last ? block_table_page(blocks, mine, b.max_blocks_per_req, kInScalar) : 0;
        const int n = min((last - pg0) / step + 1, 32);
        if (format == WARP34_KV_FORMAT_BF16 || format == WARP34_KV_FORMAT_FP8_E4M3) {
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const size_t id = (size_t)__shfl_sync(0xffffffffu, ids, i);
                take(pg0 + i * step, scored_bad_elements<false>(k_head + id * lay.k_page_stride_bytes, lay.k_token_stride_bytes, format, lane),
                     scored_bad_elements<true>(v_head + id * lay.v_page_stride_bytes, lay.v_token_stride_bytes, format, lane));
            }
            continue;
        }
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 4) {      // four pages on their way at once
            uint32_t k[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const size_t id = (size_t)__shfl_sync(0xffffffffu, ids, min(i0 + i, n - 1));
                k[i] = scored_bad_scales<false>(k_head + id * lay.k_page_stride_bytes, lay.k_token_stride_bytes, format, lane);
                v[i] = scored_bad_scales<true>(v_head + id * lay.v_page_stride_bytes, lay.v_token_stride_bytes, format, lane);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) take(pg0 + min(i0 + i, n - 1) * step, k[i], v[i]);
        }
    }
    return res;
}

// Joins what a block's warps found: k and v hold {INT_MAX, -1} before, and the block meets at a barrier on either side.
__device__ __forceinline__ void scored_bad_join(const ScoredBad& mine, int* k, int* v) {
    if ((threadIdx.x & 31) != 0) return;
    if (mine.k_first <= mine.k_last) { atomicMin(&k[0], mine.k_first); atomicMax(&k[1], mine.k_last); }
    if (mine.v_first <= mine.v_last) { atomicMin(&v[0], mine.v_first); atomicMax(&v[1], mine.v_last); }
}

// The states of W warps over parts of a row's keys (columns, maximum, mass; a mass of 0: no keys) -> the row, by one warp.
template <int W>
__device__ __forceinline__ void scored_row_join(float (*s_acc)[kHeadDim], const float* s_m, const float* s_l, bool rotated, float (&acc)[8]) {
    const int lane = threadIdx.x & 31;
    float m_tot = s_m[0], l_tot = 0.0f;
#pragma unroll 4
    for (int w = 1; w < W; ++w) m_tot = fmaxf(m_tot, s_m[w]);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
#pragma unroll 4
    for (int w = 0; w < W; ++w) {
        if (s_l[w] == 0.0f) continue;      // no keys
        const float wgt = ex2(s_m[w] - m_tot);
        l_tot += s_l[w] * wgt;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += s_acc[w][8 * lane + i] * wgt;
    }
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= rotated ? inv * 0.0625f : inv;
    if (rotated) {
        butterfly8<5>(acc, lane);
        sign8(acc, lane);
    }
}

// The same for all of a row's keys: normalised, in the natural basis, stored at `out`.
__device__ __forceinline__ void scored_row_whole(const ScoredRow& p, int req, int q_off, int q_head, void* out) {
    const int lane = threadIdx.x & 31;
    float v[8], m, l;
    scored_row_keys<4>(p, req, q_off, q_head, 0, 0x7ffffffe, 0, 1, v, m, l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const bool rotated = p.layout->v_format == WARP34_KV_FORMAT_TQ4;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= rotated ? inv * 0.0625f : inv;
    if (rotated) {
        butterfly8<5>(v, lane);
        sign8(v, lane);
    }
    store8(out, ((size_t)(p.batch->query_start_loc[req] + q_off) * p.num_q_heads + q_head) * kHeadDim, lane, p.io_bf16, v);
}

// As calls, for the chunk kernel: in line they take registers from what is around them.
__device__ __noinline__ ScoredBad scored_bad_rows_call(const ScoredRow p, int req, int kv_head, int lo, int hi, int first, int step) {
    return scored_bad_rows(p, req, kv_head, lo, hi, first, step);
}
__device__ __noinline__ void scored_row_whole_call(const ScoredRow p, int req, int q_off, int q_head, void* out) {
    scored_row_whole(p, req, q_off, q_head, out);
}

// One block of four warps per (token, q head); warp w takes every fourth group of four keys.
struct ScoredParams {
    warp34_kv_layer_layout layout;
    warp34_attention_batch batch;
    ScoreChange sc;
    const void* q_in;
    void* attn_out;
    int io_bf16, num_q_heads;
};
__global__ void __launch_bounds__(128) scored_rows_kernel(const __grid_constant__ ScoredParams p) {
    __shared__ __align__(16) float s_acc[4][kHeadDim];
    __shared__ float s_m[4], s_l[4];
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int tok = (int)(blockIdx.x / (unsigned)p.num_q_heads), q_head = (int)(blockIdx.x % (unsigned)p.num_q_heads);
    if (p.batch.valid_token_mask != nullptr && p.batch.valid_token_mask[tok] == 0) return;   // block-uniform exits
    const int req = find_request(p.batch.query_start_loc, p.batch.num_reqs, tok);
    if (req < 0 || !load_req(p.batch, req).valid) return;
    const ScoredRow row = {&p.layout, &p.batch, &p.sc, p.q_in, p.io_bf16, p.num_q_heads, p.num_q_heads / p.layout.local_kv_heads};
    float acc[8], m, l;
    scored_row_keys<4>(row, req, tok - p.batch.query_start_loc[req], q_head, 0, 0x7ffffffe, wid, 4, acc, m, l);
    *reinterpret_cast<float4*>(&s_acc[wid][8 * lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    *reinterpret_cast<float4*>(&s_acc[wid][8 * lane + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    if (lane == 0) { s_m[wid] = m; s_l[wid] = l; }
    __syncthreads();
    if (wid != 0) return;
    scored_row_join<4>(s_acc, s_m, s_l, p.layout.v_format == WARP34_KV_FORMAT_TQ4, acc);
    store8(p.attn_out, ((size_t)tok * p.num_q_heads + q_head) * kHeadDim, lane, p.io_bf16, acc);
}

static int launch_scored_rows(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch, const ScoreChange& sc,
                              const void* q_in, void* attn_out, int num_q_heads, int io_bf16) {
    const uint64_t bits = layout->k_base | layout->v_base | layout->k_page_stride_bytes | layout->k_head_stride_bytes | layout->k_token_stride_bytes |
                          layout->v_page_stride_bytes | layout->v_head_stride_bytes | layout->v_token_stride_bytes;
    const bool words = layout->k_format == WARP34_KV_FORMAT_Q8_0 || layout->k_format == WARP34_KV_FORMAT_FP8_E4M3;
    if ((bits & (words ? 3u : 1u)) != 0u) return (int)cudaErrorInvalidValue;
    const long long rows = (long long)batch->total_tokens * num_q_heads;
    if (rows > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    ScoredParams p;
    p.layout = *layout;
    p.batch = *batch;
    p.sc = sc;
    p.q_in = q_in;
    p.attn_out = attn_out;
    p.io_bf16 = io_bf16;
    p.num_q_heads = num_q_heads;
    return launch_behind(scored_rows_kernel, dim3((unsigned)rows), 128, 0, (cudaStream_t)ex->stream, p);
}

}  // namespace w34
