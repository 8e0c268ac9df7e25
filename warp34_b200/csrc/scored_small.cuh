// Scored attention of a few tokens over short contexts in one launch: a cluster of eight blocks for every (token, kv head), in fp32.
//
// The split-KV path takes three launches (plan, stream, merge) whatever the size, 19 us on a context of 317 keys.  Here the 64 warps of
// a cluster take the keys in turns; each keeps the running maximum, mass and output of the kv head's query rows, and the states meet in shared
// memory, across the cluster's blocks.  A warp's lanes hold 8 columns of every row; a key's products with GP rows are summed over the lanes
// together, half of the values leaving a lane at each step, which leaves one row's score to a lane.  One key at a time: the code then stays
// small, and a call runs most of it a few times only (four keys at a time, all unrolled, took 22 us: fetching the instructions).
// Bound by latency: about 1500 cycles a key and warp (400 instructions, two warps a scheduler), 4 us for the request's geometry, the query and the
// states' way through the cluster.
// Included by tq4_attention.cu.
#pragma once

namespace w34 {

constexpr int kSmallWarps = 8, kSmallCluster = 8;
constexpr int kSmallRow = kHeadDim + 4;    // floats of a row's state: 256 columns, maximum, mass
constexpr int kSmallAhead = 3;             // keys whose rows are on their way

struct SmallParams {
    warp34_kv_layer_layout layout;
    warp34_attention_batch batch;
    ScoreChange sc;
    const void* q_in;
    void* attn_out;
    int io_bf16, num_q_heads, gqa;
    int aligned;      // BF16 rows start on 16-byte boundaries
    int32_t* status;  // cleared, as the other paths do; may be null
};
template <int LGP> constexpr size_t small_smem_bytes() { return (size_t)(kSmallWarps + 1) * (1 << LGP) * kSmallRow * sizeof(float); }

// LGP: log2 of the rows a lane keeps, gqa rounded up to a power of two.
template <int LGP>
__global__ void __cluster_dims__(kSmallCluster, 1, 1) __launch_bounds__(kSmallWarps * 32, 1) scored_small_kernel(const __grid_constant__ SmallParams p) {
    constexpr int GP = 1 << LGP;
    constexpr int kStep = kSmallWarps * kSmallCluster;
    extern __shared__ __align__(16) float state[];      // [warp][row][256 columns, maximum, mass], then the block's by row
    __shared__ __align__(16) float s_q[GP][kHeadDim];
    __shared__ float s_centroids[16];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, rank = (int)cluster_rank();
    if (threadIdx.x < 16) s_centroids[threadIdx.x] = tq4_centroid(threadIdx.x);
    grid_dependency_wait();      // nothing above touches global memory
    grid_launch_dependents();
    if (p.status != nullptr && (blockIdx.x | blockIdx.y | blockIdx.z) == 0 && threadIdx.x == 0) *p.status = 0;
    const int tok = (int)blockIdx.y, kv_head = (int)blockIdx.z;
    // exits are the cluster's: all of them depend on the token alone
    if (p.batch.valid_token_mask != nullptr && p.batch.valid_token_mask[tok] == 0) return;
    const int req = find_request(p.batch.query_start_loc, p.batch.num_reqs, tok);
    if (req < 0) return;
    const ReqGeom g = load_req(p.batch, req);
    if (!g.valid) return;
    const int q_off = tok - g.q_start, q_pos = g.ctx_before + q_off;
    const int lo = row_first_key<true>(p.batch, p.sc, g, q_off), hi = row_last_key<true>(p.batch, p.sc, g, q_off);
    const int k_format = p.layout.k_format, v_format = p.layout.v_format;
    const int32_t* blocks = p.batch.block_tables + (size_t)req * p.batch.max_blocks_per_req;
    const uint8_t* k_head = (const uint8_t*)(uintptr_t)p.layout.k_base + (size_t)kv_head * p.layout.k_head_stride_bytes;
    const uint8_t* v_head = (const uint8_t*)(uintptr_t)p.layout.v_base + (size_t)kv_head * p.layout.v_head_stride_bytes;
    const long long keys = (long long)hi - lo + 1;

    // The rows of a warp's next keys are on their way while it works on one, and the page of the key behind those.
    ScoredRaw k_ahead[kSmallAhead] = {}, v_ahead[kSmallAhead] = {};
    auto page_of = [&](long long n) { return n < keys ? block_table_page(blocks, (lo + (int)n) >> 4, p.batch.max_blocks_per_req, kInScalar) : 0; };
    auto load = [&](ScoredRaw& k, ScoredRaw& v, long long n, int page) {
        if (n >= keys) return;
        const size_t off = (size_t)((lo + (int)n) & 15);
        scored_load(k, k_head + (size_t)page * p.layout.k_page_stride_bytes + off * p.layout.k_token_stride_bytes, k_format, lane, p.aligned);
        scored_load(v, v_head + (size_t)page * p.layout.v_page_stride_bytes + off * p.layout.v_token_stride_bytes, v_format, lane, p.aligned);
    };
    long long n = rank * kSmallWarps + wid;
    int page;
    {
        int first[kSmallAhead];
#pragma unroll
        for (int a = 0; a < kSmallAhead; ++a) first[a] = page_of(n + a * kStep);
        page = page_of(n + kSmallAhead * kStep);
#pragma unroll
        for (int a = 0; a < kSmallAhead; ++a) load(k_ahead[a], v_ahead[a], n + a * kStep, first[a]);
    }
    // query rows, in the stored basis and scaled: a row a warp
    for (int r = wid; r < GP; r += kSmallWarps) {
        float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (r < p.gqa) {
            load8(p.q_in, ((size_t)tok * p.num_q_heads + kv_head * p.gqa + r) * kHeadDim, lane, p.io_bf16, q);
            float scale = p.batch.sm_scale * 1.4426950408889634f;
            if (k_format == WARP34_KV_FORMAT_TQ4) {
                sign8(q, lane);
                butterfly8<5>(q, lane);
                scale *= 0.0625f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] *= scale;
        }
        *reinterpret_cast<float4*>(&s_q[r][8 * lane]) = make_float4(q[0], q[1], q[2], q[3]);
        *reinterpret_cast<float4*>(&s_q[r][8 * lane + 4]) = make_float4(q[4], q[5], q[6], q[7]);
    }
    __syncthreads();
    float q[GP][8], acc[GP][8];
#pragma unroll
    for (int r = 0; r < GP; ++r) {
        const float4 a = *reinterpret_cast<const float4*>(&s_q[r][8 * lane]), b = *reinterpret_cast<const float4*>(&s_q[r][8 * lane + 4]);
        q[r][0] = a.x; q[r][1] = a.y; q[r][2] = a.z; q[r][3] = a.w; q[r][4] = b.x; q[r][5] = b.y; q[r][6] = b.z; q[r][7] = b.w;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r][i] = 0.0f;
    }
    const int my_row = lane >> (5 - LGP);      // the row whose score ends in this lane
    const float slope = my_row < p.gqa ? row_slope(p.sc, kv_head * p.gqa + my_row) : 0.0f;
    float m = -1e30f, l = 0.0f;      // of my_row
    const auto centroid = [&](uint32_t code) { return s_centroids[code]; };
#pragma unroll 1
    for (; n < keys; n += kStep) {
        const ScoredRaw kr = k_ahead[0], vr = v_ahead[0];
#pragma unroll
        for (int a = 0; a + 1 < kSmallAhead; ++a) {
            k_ahead[a] = k_ahead[a + 1];
            v_ahead[a] = v_ahead[a + 1];
        }
        load(k_ahead[kSmallAhead - 1], v_ahead[kSmallAhead - 1], n + kSmallAhead * kStep, page);
        page = page_of(n + (kSmallAhead + 1) * kStep);
        float x[8], s[GP];
        scored_values(kr, k_format, centroid, x);
#pragma unroll
        for (int r = 0; r < GP; ++r) {
            s[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[r] = __fmaf_rn(q[r][i], x[i], s[r]);
        }
        const float t = changed_score(p.sc, scored_sums(s, lane), slope, (float)(q_pos - (lo + (int)n)));
        const float m_new = fmaxf(m, t), alpha = ex2(m - m_new), w = ex2(t - m_new);
        m = m_new;
        l = l * alpha + w;
        if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
            for (int r = 0; r < GP; ++r) {
                const float a = __shfl_sync(0xffffffffu, alpha, r << (5 - LGP));
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[r][i] *= a;
            }
        }
        scored_values(vr, v_format, centroid, x);
#pragma unroll
        for (int r = 0; r < GP; ++r) {
            const float wr = __shfl_sync(0xffffffffu, w, r << (5 - LGP));
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r][i] = __fmaf_rn(wr, x[i], acc[r][i]);
        }
    }
    float* mine = state + (size_t)wid * GP * kSmallRow;
#pragma unroll
    for (int r = 0; r < GP; ++r) {
        float* row = mine + r * kSmallRow;
#pragma unroll
        for (int i = 0; i < 8; i += 2) *reinterpret_cast<float2*>(row + 8 * lane + i) = make_float2(acc[r][i], acc[r][i + 1]);
        const float mr = __shfl_sync(0xffffffffu, m, r << (5 - LGP)), lr = __shfl_sync(0xffffffffu, l, r << (5 - LGP));
        if (lane == 0) {
            row[kHeadDim] = mr;
            row[kHeadDim + 1] = lr;
        }
    }
    __syncthreads();
    // ---- warp r combines the block's states of row r; block r then the eight blocks' ---------------------------------------
    // Combination of eight states `from(w)` (addresses of rows of kSmallRow floats), by one warp; a state without keys holds zeros.
    auto combine = [&](auto from, float (&v)[8], float& m_all, float& l_all) {
        float4 a[kSmallWarps], b[kSmallWarps];      // all on their way before the first is used
        float2 ml[kSmallWarps];
#pragma unroll
        for (int w = 0; w < kSmallWarps; ++w) {
            const uint32_t at = from(w);
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[w].x), "=f"(ml[w].y) : "r"(at + 4u * kHeadDim) : "memory");
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a[w].x), "=f"(a[w].y), "=f"(a[w].z), "=f"(a[w].w) : "r"(at + 32u * lane) : "memory");
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(b[w].x), "=f"(b[w].y), "=f"(b[w].z), "=f"(b[w].w) : "r"(at + 32u * lane + 16u) : "memory");
        }
        m_all = -1e30f;
        l_all = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < kSmallWarps; ++w) m_all = fmaxf(m_all, ml[w].y != 0.0f ? ml[w].x : -1e30f);
#pragma unroll
        for (int w = 0; w < kSmallWarps; ++w) {
            const float f = ml[w].y != 0.0f ? ex2(ml[w].x - m_all) : 0.0f;
            l_all = __fmaf_rn(ml[w].y, f, l_all);
            v[0] = __fmaf_rn(a[w].x, f, v[0]); v[1] = __fmaf_rn(a[w].y, f, v[1]); v[2] = __fmaf_rn(a[w].z, f, v[2]); v[3] = __fmaf_rn(a[w].w, f, v[3]);
            v[4] = __fmaf_rn(b[w].x, f, v[4]); v[5] = __fmaf_rn(b[w].y, f, v[5]); v[6] = __fmaf_rn(b[w].z, f, v[6]); v[7] = __fmaf_rn(b[w].w, f, v[7]);
        }
    };
    static_assert(kSmallWarps == kSmallCluster, "eight states either time");
    const uint32_t states = (uint32_t)__cvta_generic_to_shared(state);
    float* combined = state + (size_t)kSmallWarps * GP * kSmallRow;      // [row]
    if (wid < p.gqa) {
        float v[8], m_all, l_all;
        combine([&](int w) { return states + 4u * (uint32_t)((w * GP + wid) * kSmallRow); }, v, m_all, l_all);
        float* row = combined + wid * kSmallRow;
        *reinterpret_cast<float4*>(row + 8 * lane) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + 8 * lane + 4) = make_float4(v[4], v[5], v[6], v[7]);
        if (lane == 0) *reinterpret_cast<float2*>(row + kHeadDim) = make_float2(m_all, l_all);
    }
    cluster_sync_all();
    if (wid == 0 && rank < p.gqa) {
        float v[8], m_all, l_all;
        const uint32_t row = states + 4u * (uint32_t)((kSmallWarps * GP + rank) * kSmallRow);
        combine([&](int w) { return map_to_rank(row, (uint32_t)w); }, v, m_all, l_all);
        const bool rotated = v_format == WARP34_KV_FORMAT_TQ4;
        const float inv = (l_all == 0.0f ? 0.0f : 1.0f / l_all) * (rotated ? 0.0625f : 1.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= inv;
        if (rotated) {
            butterfly8<5>(v, lane);
            sign8(v, lane);
        }
        store8(p.attn_out, ((size_t)tok * p.num_q_heads + kv_head * p.gqa + rank) * kHeadDim, lane, p.io_bf16, v);
    }
    cluster_sync_all();      // no block leaves while another reads its states
}

// Which calls: up to 8 rows per kv head, and clusters that are served at once (of more than two rows a block fills its SM: fewer than 16 clusters
// fit) up to 1024 keys, or in two rounds up to 256.  Measured, this kernel / the split-KV path, us a call with a cold L2: one token of 24 / 4 heads over
// 16 / 300 / 1000 / 2000 TQ4 keys 10 / 23, 14 / 41, 23 / 39, 35 / 35; BF16 10 / 23, 14 / 33, 21 / 33, 33 / 29; FP8 10 / 21, 14 / 23, 23 / 25, 35 / 23.
// Four tokens (16 clusters, two rounds) over 100 / 300 / 1000 FP8 keys 18 / 23, 23 / 25, 39 / 25; the same on 4 / 4 heads 10 / 25, 12 / 25, 21 / 27.
static bool takes_small(const warp34_kv_layer_layout* l, const warp34_attention_batch* b, int num_q_heads) {
    const long long keys = b->max_seq_len > 0 ? (long long)b->max_seq_len : (long long)b->max_blocks_per_req * kPageTokens;
    const long long clusters = (long long)b->total_tokens * l->local_kv_heads, gqa = num_q_heads / l->local_kv_heads;
    return gqa <= 8 && ((clusters <= (gqa <= 2 ? 24 : 12) && keys <= 1024) || (clusters <= 24 && keys <= 256));
}
static int launch_scored_small(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch, const ScoreChange& sc,
                               const void* q_in, void* attn_out, int num_q_heads, int io_bf16) {
    const uint64_t bits = layout->k_base | layout->v_base | layout->k_page_stride_bytes | layout->k_head_stride_bytes | layout->k_token_stride_bytes |
                          layout->v_page_stride_bytes | layout->v_head_stride_bytes | layout->v_token_stride_bytes;
    const bool words = layout->k_format == WARP34_KV_FORMAT_Q8_0 || layout->k_format == WARP34_KV_FORMAT_FP8_E4M3;
    if ((bits & (words ? 3u : 1u)) != 0u) return (int)cudaErrorInvalidValue;
    SmallParams p;
    p.layout = *layout;
    p.batch = *batch;
    p.sc = sc;
    p.q_in = q_in;
    p.attn_out = attn_out;
    p.io_bf16 = io_bf16;
    p.num_q_heads = num_q_heads;
    p.gqa = num_q_heads / layout->local_kv_heads;
    p.aligned = (bits & 15u) == 0u ? 1 : 0;
    p.status = ex->scratch_ptr != 0 && (ex->scratch_ptr & 3u) == 0 && ex->scratch_size >= sizeof(PlanHeader) ? reinterpret_cast<int32_t*>((uintptr_t)ex->scratch_ptr) : nullptr;
    const dim3 grid(kSmallCluster, (unsigned)batch->total_tokens, (unsigned)layout->local_kv_heads);
    cudaStream_t st = (cudaStream_t)ex->stream;
    if (p.gqa == 1) return launch_behind(scored_small_kernel<0>, grid, kSmallWarps * 32, small_smem_bytes<0>(), st, p);
    if (p.gqa == 2) return launch_behind(scored_small_kernel<1>, grid, kSmallWarps * 32, small_smem_bytes<1>(), st, p);
    if (p.gqa <= 4) return launch_behind(scored_small_kernel<2>, grid, kSmallWarps * 32, small_smem_bytes<2>(), st, p);
    return launch_behind(scored_small_kernel<3>, grid, kSmallWarps * 32, small_smem_bytes<3>(), st, p);
}

}  // namespace w34
