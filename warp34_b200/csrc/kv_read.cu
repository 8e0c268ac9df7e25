// Cached rows read back as 16-bit values: the inverse of the append, for every layer format.
//
//   TQ4        x = s * H y / 16,  y[c] = d[c >> 7] * centroid[code[c]]     (s sign diagonal, H the 256-point Walsh-Hadamard matrix)
//   FP8 E4M3   x[c] = d[c >> 7] * code[c]          Q8_0   x[c] = d[c >> 6] * code[c]          BF16   x = row
//
// in fp32, rounded once to the output type.
//
// A warp holds a row (and, where there are tokens enough, four rows of neighbouring heads on their way at once).  TQ4: column 16 a + b of
// the row is element (b, a) of a 16 x 16 matrix, and the transform a product from either side, both on the tensor cores
// (mma.sync m16n8k16, fp32 accumulators) with a matrix of +-1:
//     Z = (H / 256) (16 X),  U = Z (1 x H8),  Y = d0 U0 +- d1 U1
// with U0, U1 the 8-point transforms of the two halves of Z's columns, which have a scale each, and the last level, where they meet, in fp32.
// X comes as fp16 value and residual from a table by code byte (22 bits of a centroid), Z is split the same way: eight products a row.
// The accumulators of the first are the A fragments of the second as they lie in the lanes; columns of the first +-1 matrix are ordered so
// that a lane's elements are four neighbouring columns (two code bytes).  The rounded row passes through shared memory (stmatrix,
// transposed), so that a lane stores 16 bytes.  (With movmatrix instead of that and 8 bytes a lane 124 instructions a row, 23 of them on the shared-memory pipe instead of 12.)
// (Eight lanes to a row, the transform in packed fp32 arithmetic and its columns changing lanes through shared memory: 67 us instead of
// 52 for 35065 tokens of 4 heads, at 40 shared-memory wavefronts and 168 instructions a row.)
// What that is off by: an element of Z 2^-25 twice, its sums and X 2^-24 more; U sums eight of them, Y both halves with their scales: 18 x 2^-24
// (|d0| + |d1|) at most, 2^-24 (|d0| + |d1|) in the root mean square of independent roundings, where a row's values are about (|d0| + |d1|) / 32.
// Bound by instruction issue: 119 a row, two thirds of the slots with 24 warps an SM; HBM is at 0.54 of the copy rate.  The same 35065 tokens
// of FP8, Q8_0 and BF16 rows take 45.5, 44.4 and 51.0 us (0.74, 0.77 and 0.87 of it).  The rows of a warp's next token are on their way while it computes (57 instead of 61 us with a cold L2; with the
// registers of four blocks an SM instead of three they spill).
#include "tq4_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

namespace w34 {

constexpr int kReadWarps = 8;
constexpr int kReadTq4Blocks = 3;              // resident blocks an SM that a grid is sized for
constexpr int kReadRows = 4;                   // rows of a warp on their way at once: heads of one token
constexpr int kReadTableBytes = 256 * 128;     // byte -> (value pair, residual pair), 16 copies

struct ReadParams {
    warp34_kv_layer_layout layout;
    warp34_attention_batch batch;
    uint16_t* out[2];           // K, V
    long long stride[2];        // elements
    int first, sides;           // 0: K first; how many of the two are read
    int aligned;                // output rows start on 16-byte boundaries
    int rows_aligned;           // BF16 rows do
    int tokens_per_warp;
};

template <bool BF16>
__device__ __forceinline__ uint32_t read_narrow(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void read_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void read_mma_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void read_mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ void read_mma8_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
__device__ __forceinline__ uint32_t read_half2(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// a and b as fp16 pairs of values and of residuals.  The value is cut off to fp16's 11 bits, not rounded (one instruction), and exact as fp16 from
// 2^-14 up; the residual is below 2^-10 of it.  Elements of Z are 1/64 and less than 0.17 in magnitude, so residuals, and values below 2^-14, are in
// the range of fp16's fixed steps of 2^-24: each is off by 2^-25 at most.
__device__ __forceinline__ void read_split(float a, float b, uint32_t& value, uint32_t& residual) {
    const float va = __uint_as_float(__float_as_uint(a) & 0xffffe000u), vb = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
    value = read_half2(va, vb);
    const Two rest = fma_two(two_of(va, vb), two_of(-1.0f, -1.0f), two_of(a, b));
    residual = read_half2(first_of(rest), second_of(rest));
}
// Entries (i, j0), (i, j1) of the 16-point Walsh-Hadamard matrix times `scale`, as an fp16 pair.
__device__ __forceinline__ uint32_t read_hadamard(int i, int j0, int j1, float scale) {
    return read_half2((__popc(i & j0) & 1) ? -scale : scale, (__popc(i & j1) & 1) ? -scale : scale);
}
// Page and offset of token `tok`, or a negative page: the token takes no part.
__device__ __forceinline__ int read_place(const ReadParams& p, int tok, int& off) {
    const warp34_attention_batch& b = p.batch;
    if (b.valid_token_mask != nullptr && b.valid_token_mask[tok] == 0) return -1;
    if (b.write_slot_mapping != nullptr && b.valid_req_mask == nullptr) {
        if (tok < b.query_start_loc[0] || tok >= b.query_start_loc[b.num_reqs]) return -1;
    }
    const bool by_slot = b.write_slot_mapping != nullptr;
    int r = 0;
    if (!by_slot || b.valid_req_mask != nullptr) {
        r = find_request(b.query_start_loc, b.num_reqs, tok);
        if (r < 0 || (b.valid_req_mask != nullptr && b.valid_req_mask[r] == 0)) return -1;
    }
    int page;
    if (by_slot) {
        const int slot = b.write_slot_mapping[tok];
        if (slot < 0) return -1;
        page = slot >> 4;
        off = slot & 15;
    } else {
        const int q_len = b.query_start_loc[r + 1] - b.query_start_loc[r];
        const int pos = (b.context_lens_before != nullptr ? b.context_lens_before[r] : b.seq_lens_after[r] - q_len) + (tok - b.query_start_loc[r]);
        if (pos < 0 || (pos >> 4) >= b.max_blocks_per_req) return -1;
        page = block_table_page(b.block_tables + (size_t)r * b.max_blocks_per_req, pos >> 4, b.max_blocks_per_req, kInRead);
        off = pos & 15;
    }
    return pool_page(page, kInRead);
}
__device__ __forceinline__ const uint8_t* read_row(const ReadParams& p, int page, int off, int head, int side) {
    const warp34_kv_layer_layout& l = p.layout;
    const uint64_t at = side == 0 ? l.k_base + (uint64_t)page * l.k_page_stride_bytes + (uint64_t)head * l.k_head_stride_bytes + (uint64_t)off * l.k_token_stride_bytes
                                  : l.v_base + (uint64_t)page * l.v_page_stride_bytes + (uint64_t)head * l.v_head_stride_bytes + (uint64_t)off * l.v_token_stride_bytes;
    return reinterpret_cast<const uint8_t*>((uintptr_t)at);
}

// The tokens of a warp are neighbours, an equal share for every warp of the grid.  Its lanes look up 32 of their rows at once: looked up
// one by one, a token's place cost as much as one and a half of its rows.
struct ReadShare {
    int first, end;
    __device__ __forceinline__ explicit ReadShare(const ReadParams& p) {
        const long long w = (long long)blockIdx.x * kReadWarps + (threadIdx.x >> 5), per = p.tokens_per_warp;
        first = (int)min(w * per, (long long)p.batch.total_tokens);
        end = (int)min((w + 1) * per, (long long)p.batch.total_tokens);
    }
};
// Address of the row of token first + lane, or 0.
__device__ __forceinline__ uint64_t read_rows_of(const ReadParams& p, int first, int end, int head, int side) {
    const int tok = first + (int)(threadIdx.x & 31);
    int off = 0;
    const int page = tok < end ? read_place(p, tok, off) : -1;
    return page < 0 ? 0 : (uint64_t)(uintptr_t)read_row(p, page, off, head, side);
}

// blockIdx.y: side x group of ROWS heads.
template <bool BF16, int ROWS>
__global__ void __launch_bounds__(kReadWarps * 32, kReadTq4Blocks) kv_read_tq4_kernel(const __grid_constant__ ReadParams p) {
    __shared__ __align__(128) uint8_t table[kReadTableBytes];
    __shared__ __align__(128) uint8_t turns[512 * kReadWarps];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3;
    {      // entry `threadIdx.x`; centroids x 16 (0.13 to 2.7), so that 2^-25, the most by which their residuals are off, is 2^-22 of the smallest
        const float c0 = 16.0f * tq4_centroid(threadIdx.x & 15), c1 = 16.0f * tq4_centroid(threadIdx.x >> 4);
        const uint32_t hi = read_half2(c0, c1);
        const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        const uint2 e = make_uint2(hi, read_half2(c0 - hf.x, c1 - hf.y));
        static_assert(kReadWarps * 32 == 256, "one entry per thread");
#pragma unroll
        for (int i = 0; i < 16; ++i) *reinterpret_cast<uint2*>(table + threadIdx.x * 128 + ((i + threadIdx.x) & 15) * 8) = e;
    }
    // k position 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of a product <-> b = 4 t .. 4 t + 3
    auto order = [](int m) { return 4 * ((m & 7) >> 1) + (m & 1) + 2 * (m >> 3); };
    uint32_t ha[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {      // A fragment: rows gid, gid + 8, k 2 tig (+ 8)
        const int m = gid + 8 * (i & 1), k = 2 * tig + 8 * (i >> 1);
        ha[i] = read_hadamard(m, order(k), order(k + 1), 1.0f / 256.0f);
    }
    const uint32_t hb = read_hadamard(gid, 2 * tig, 2 * tig + 1, 1.0f);
    uint32_t sign[4];      // of columns 8 lane .. + 7, as the sign bits of packed pairs
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t m = c_sign_mask[lane >> 2] >> (8 * (lane & 3) + 2 * k);
        sign[k] = ((m & 1u) << 15) | ((m & 2u) << 30);
    }
    grid_dependency_wait();      // nothing above touches global memory
    grid_launch_dependents();
    __syncthreads();
    const uint32_t copy = 8u * (uint32_t)(lane & 15);
    const int heads = p.layout.local_kv_heads, groups = (heads + ROWS - 1) / ROWS;
    const int side = p.first + (int)blockIdx.y / groups, head0 = (int)blockIdx.y % groups * ROWS;
    const uint64_t head_stride = side == 0 ? p.layout.k_head_stride_bytes : p.layout.v_head_stride_bytes;
    const int n_rows = min(ROWS, heads - head0);
    // The finished row passes through 512 bytes of this warp's: 16-byte chunk c (columns 8 c .. + 7) at place c ^ (c >> 3 & 1), free of bank
    // conflicts for the matrices' rows (every other chunk) and for the lanes' chunks.
    const uint32_t turn = (uint32_t)__cvta_generic_to_shared(turns) + 512u * (uint32_t)wid;
    const int m_row = 8 * (lane >> 4) + (lane & 7), m_chunk = 2 * m_row + ((lane >> 3) & 1);      // matrix lane / 8: a' 8 (lane / 16) .., b' 8 (lane / 8 % 2) ..
    const uint32_t turn_in = turn + 16u * (uint32_t)(m_chunk ^ ((m_chunk >> 3) & 1)), turn_out = turn + 16u * (uint32_t)(lane ^ ((lane >> 3) & 1));
    const ReadShare share(p);
    uint64_t rows = 0;
    uint16_t* dst = p.out[side] + (size_t)share.first * (size_t)p.stride[side] + (head0 * kHeadDim + 8 * lane);
    // Codes and scales (fp16 bits) of a token's rows; those of the next token are on their way while a token's are computed.
    struct Raw { uint32_t codes[ROWS][2], scales[ROWS][2]; };
    auto load = [&](Raw& raw, uint64_t at) {
        const uint8_t* row = reinterpret_cast<const uint8_t*>((uintptr_t)at);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (at == 0 || (ROWS > 1 && i >= n_rows)) break;
            const uint8_t* mine = row + (2 + 8 * gid + 2 * tig);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                raw.codes[i][h] = *reinterpret_cast<const uint16_t*>(mine + kTq4BlockBytes * h);
                raw.scales[i][h] = *reinterpret_cast<const uint16_t*>(row + kTq4BlockBytes * h);
            }
            row += head_stride;
        }
    };
    uint64_t at_next = 0;
    Raw next = {};
    if (share.first < share.end) {
        rows = read_rows_of(p, share.first, share.end, head0, side);
        at_next = __shfl_sync(0xffffffffu, rows, 0);
        load(next, at_next);
    }
#pragma unroll 1
    for (int t = share.first; t < share.end; ++t, dst += p.stride[side]) {
        const uint64_t at = at_next;
        const Raw raw = next;
        const int k32 = (t + 1 - share.first) & 31;
        if (k32 == 0 && t + 1 < share.end) rows = read_rows_of(p, t + 1, share.end, head0, side);
        at_next = t + 1 < share.end ? __shfl_sync(0xffffffffu, rows, k32) : 0;
        load(next, at_next);
        if (at == 0) continue;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (ROWS > 1 && i >= n_rows) break;
            float u[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {      // the half with scale d[h]: a = 8 h + n
                const uint2 e0 = *reinterpret_cast<const uint2*>(table + (((raw.codes[i][h] << 7) & 0x7f80u) | copy));
                const uint2 e1 = *reinterpret_cast<const uint2*>(table + (((raw.codes[i][h] >> 1) & 0x7f80u) | copy));
                float z[4];
                read_mma_zero(z, ha[0], ha[1], ha[2], ha[3], e0.x, e1.x);
                read_mma(z, ha[0], ha[1], ha[2], ha[3], e0.y, e1.y);
                uint32_t v0, v1, r0, r1;
                read_split(z[0], z[1], v0, r0);
                read_split(z[2], z[3], v1, r1);
                read_mma8_zero(u[h], v0, v1, hb);
                read_mma8(u[h], r0, r1, hb);
            }
            const float d0 = __half2float(__ushort_as_half((unsigned short)raw.scales[i][0])), d1 = __half2float(__ushort_as_half((unsigned short)raw.scales[i][1]));
            uint32_t w[2][2];      // matrices (a' 8 n .., b' 8 m ..)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const Two low = mul_two(two_of(u[0][2 * m], u[0][2 * m + 1]), two_of(d0, d0)), high = two_of(u[1][2 * m], u[1][2 * m + 1]);
                const Two sum = fma_two(high, two_of(d1, d1), low), difference = fma_two(high, two_of(-d1, -d1), low);
                w[0][m] = read_narrow<BF16>(first_of(sum), second_of(sum));
                w[1][m] = read_narrow<BF16>(first_of(difference), second_of(difference));
            }
            __syncwarp();      // the row before has been read
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                         ::"r"(turn_in), "r"(w[0][0]), "r"(w[0][1]), "r"(w[1][0]), "r"(w[1][1]) : "memory");
            __syncwarp();
            uint32_t r[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(turn_out) : "memory");
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k] ^= sign[k];
            uint16_t* to = dst + i * kHeadDim;
            if (p.aligned) {
                *reinterpret_cast<uint4*>(to) = make_uint4(r[0], r[1], r[2], r[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) { to[2 * k] = (uint16_t)r[k]; to[2 * k + 1] = (uint16_t)(r[k] >> 16); }
            }
        }
    }
}

// Rows that are not rotated: lane l holds columns 8 l .. + 7.
template <bool BF16, int ROWS>
__global__ void __launch_bounds__(kReadWarps * 32) kv_read_plain_kernel(const __grid_constant__ ReadParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int heads = p.layout.local_kv_heads, groups = (heads + ROWS - 1) / ROWS;
    const int side = p.first + (int)blockIdx.y / groups, head0 = (int)blockIdx.y % groups * ROWS;
    const uint64_t head_stride = side == 0 ? p.layout.k_head_stride_bytes : p.layout.v_head_stride_bytes;
    const int format = side == 0 ? p.layout.k_format : p.layout.v_format;
    const ReadShare share(p);
    uint64_t rows = 0;
    uint16_t* dst = p.out[side] + (size_t)share.first * (size_t)p.stride[side] + (head0 * kHeadDim + 8 * lane);
#pragma unroll 1
    for (int t = share.first; t < share.end; ++t, dst += p.stride[side]) {
        const int k32 = (t - share.first) & 31;
        if (k32 == 0) rows = read_rows_of(p, t, share.end, head0, side);
        const uint8_t* row = reinterpret_cast<const uint8_t*>((uintptr_t)__shfl_sync(0xffffffffu, rows, k32));
        if (row == nullptr) continue;
        uint32_t raw[ROWS][4];
        float d[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (ROWS > 1 && head0 + i >= heads) break;
            const uint8_t* r = row + (size_t)i * head_stride;
            if (format == WARP34_KV_FORMAT_BF16) {
                const uint16_t* src = reinterpret_cast<const uint16_t*>(r) + 8 * lane;
                if (p.rows_aligned) {
                    const uint4 q = *reinterpret_cast<const uint4*>(src);
                    raw[i][0] = q.x; raw[i][1] = q.y; raw[i][2] = q.z; raw[i][3] = q.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) raw[i][k] = (uint32_t)src[2 * k] | ((uint32_t)src[2 * k + 1] << 16);
                }
            } else {
                const bool fp8 = format == WARP34_KV_FORMAT_FP8_E4M3;
                const uint32_t* src = reinterpret_cast<const uint32_t*>(r + (fp8 ? 8 * lane : 68 * (lane >> 3) + 4 + 8 * (lane & 7)));
                raw[i][0] = src[0];
                raw[i][1] = src[1];
                d[i] = *reinterpret_cast<const float*>(r + (fp8 ? kHeadDim + 4 * (lane >> 4) : 68 * (lane >> 3)));
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (ROWS > 1 && head0 + i >= heads) break;
            uint32_t w[4];
            if (format == WARP34_KV_FORMAT_BF16) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    w[k] = BF16 ? raw[i][k] : read_narrow<false>(__uint_as_float(raw[i][k] << 16), __uint_as_float(raw[i][k] & 0xffff0000u));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t two = raw[i][k >> 1] >> (16 * (k & 1));
                    float a, b;
                    if (format == WARP34_KV_FORMAT_FP8_E4M3) {
                        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffffu), __NV_E4M3);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                        a = f.x;
                        b = f.y;
                    } else {
                        a = (float)(int8_t)(two & 0xffu);
                        b = (float)(int8_t)((two >> 8) & 0xffu);
                    }
                    w[k] = read_narrow<BF16>(d[i] * a, d[i] * b);
                }
            }
            uint16_t* to = dst + (size_t)i * kHeadDim;
            if (p.aligned) {
                *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) { to[2 * k] = (uint16_t)w[k]; to[2 * k + 1] = (uint16_t)(w[k] >> 16); }
            }
        }
    }
}

W34_BOUNDS_HOST_HOOKS(read)

static int read_sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
    return sms;
}

template <bool BF16>
static int launch_kv_read(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch, void* k_out, void* v_out,
                          int k_row_stride, int v_row_stride) {
    if (ex == nullptr || layout == nullptr || batch == nullptr || (k_out == nullptr && v_out == nullptr) || batch->total_tokens < 0 ||
        layout->local_kv_heads <= 0) {
        return (int)cudaErrorInvalidValue;
    }
    if (batch->total_tokens == 0) return 0;
    const warp34_kv_layer_layout& l = *layout;
    auto unrotated = [&](int f) { return f == WARP34_KV_FORMAT_Q8_0 || f == WARP34_KV_FORMAT_FP8_E4M3; };
    const bool identity = l.k_transform == WARP34_KV_TRANSFORM_IDENTITY && l.v_transform == WARP34_KV_TRANSFORM_IDENTITY;
    const bool tq4 = l.k_format == WARP34_KV_FORMAT_TQ4 && l.v_format == WARP34_KV_FORMAT_TQ4 &&
                     l.k_transform == WARP34_KV_TRANSFORM_RADEMACHER_WHT256 && l.v_transform == WARP34_KV_TRANSFORM_RADEMACHER_WHT256;
    const bool eight = identity && unrotated(l.k_format) && unrotated(l.v_format);
    const bool bf16 = identity && l.k_format == WARP34_KV_FORMAT_BF16 && l.v_format == WARP34_KV_FORMAT_BF16;
    if (l.head_dim != kHeadDim || l.block_size != kPageTokens || !(tq4 || eight || bf16)) return (int)cudaErrorNotSupported;
    const int cols = l.local_kv_heads * kHeadDim;
    if ((k_out != nullptr && k_row_stride < cols) || (v_out != nullptr && v_row_stride < cols) || l.k_base == 0 || l.v_base == 0 ||
        batch->num_reqs <= 0 || batch->query_start_loc == nullptr ||
        (batch->write_slot_mapping == nullptr && (batch->block_tables == nullptr || batch->max_blocks_per_req <= 0 ||
                                                  (batch->context_lens_before == nullptr && batch->seq_lens_after == nullptr)))) {
        return (int)cudaErrorInvalidValue;
    }
    const uint64_t bits = l.k_base | l.v_base | l.k_page_stride_bytes | l.v_page_stride_bytes | l.k_head_stride_bytes | l.v_head_stride_bytes |
                          l.k_token_stride_bytes | l.v_token_stride_bytes;
    if ((bits & (eight ? 3u : 1u)) != 0u || ((((uintptr_t)k_out) | ((uintptr_t)v_out)) & 1u) != 0u) return (int)cudaErrorInvalidValue;
    ReadParams p;
    p.layout = l;
    p.batch = *batch;
    p.out[0] = static_cast<uint16_t*>(k_out);
    p.out[1] = static_cast<uint16_t*>(v_out);
    p.stride[0] = k_row_stride;
    p.stride[1] = v_row_stride;
    p.first = k_out != nullptr ? 0 : 1;
    p.sides = (k_out != nullptr ? 1 : 0) + (v_out != nullptr ? 1 : 0);
    p.aligned = ((((uintptr_t)k_out) | ((uintptr_t)v_out)) & 15u) == 0u && (k_out == nullptr || k_row_stride % 8 == 0) && (v_out == nullptr || v_row_stride % 8 == 0);
    p.rows_aligned = (bits & 15u) == 0u;
    const int sms = read_sm_count();
    const int cols_y = p.sides * l.local_kv_heads;      // rows of a token
    // Four heads a warp, their loads in flight together, where that still leaves every SM several blocks.
    const bool wide = (long long)batch->total_tokens * cols_y >= 32ll * kReadWarps * sms;
    const int rows_y = wide ? p.sides * ((l.local_kv_heads + kReadRows - 1) / kReadRows) : cols_y;
    if (rows_y > 65535) return (int)cudaErrorInvalidValue;
    const long long needed = ((long long)batch->total_tokens + kReadWarps - 1) / kReadWarps;
    const long long resident = ((long long)sms * (tq4 ? kReadTq4Blocks : 8)) / rows_y > 0 ? ((long long)sms * (tq4 ? kReadTq4Blocks : 8)) / rows_y : 1;
    const dim3 grid((unsigned)(needed < resident ? needed : resident), (unsigned)rows_y);
    p.tokens_per_warp = (int)(((long long)batch->total_tokens + (long long)grid.x * kReadWarps - 1) / ((long long)grid.x * kReadWarps));
    cudaStream_t st = (cudaStream_t)ex->stream;
    if (!tq4) {
        return wide ? launch_behind(kv_read_plain_kernel<BF16, kReadRows>, grid, kReadWarps * 32, 0, st, p)
                    : launch_behind(kv_read_plain_kernel<BF16, 1>, grid, kReadWarps * 32, 0, st, p);
    }
    return wide ? launch_behind(kv_read_tq4_kernel<BF16, kReadRows>, grid, kReadWarps * 32, 0, st, p)
                : launch_behind(kv_read_tq4_kernel<BF16, 1>, grid, kReadWarps * 32, 0, st, p);
}

}  // namespace w34

extern "C" int warp34_kv_cache_read_f16(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch, void* k_out,
                                        void* v_out, int k_row_stride, int v_row_stride) {
    return w34::launch_kv_read<false>(ex, layout, batch, k_out, v_out, k_row_stride, v_row_stride);
}
extern "C" int warp34_kv_cache_read_bf16(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch, void* k_out,
                                         void* v_out, int k_row_stride, int v_row_stride) {
    return w34::launch_kv_read<true>(ex, layout, batch, k_out, v_out, k_row_stride, v_row_stride);
}
