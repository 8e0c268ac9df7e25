// Cached rows read back as 16-bit values: the inverse of the append, for every layer format.
//
//   TQ4        x = s * H y / 16,  y[c] = d[c >> 7] * centroid[code[c]]     (s sign diagonal, H the 256-point Walsh-Hadamard matrix)
//   FP8 E4M3   x[c] = d[c >> 7] * code[c]          Q8_0   x[c] = d[c >> 6] * code[c]          BF16   x = row
//
// in fp32, rounded once to the output type.
//
// Eight lanes hold a row, a warp four rows of neighbouring tokens.  The output is three quarters of the bytes, so it decides the
// layout: a lane ends with 16-byte chunks j + 8 i of its row, eight lanes write whole 128-byte lines.  TQ4 rows start in the other
// layout, quads (4 columns, 2 bytes of codes): there five levels of the transform are register arithmetic, the columns then
// change lanes through shared memory once, and the other three are register arithmetic again.  Both scales of a row meet in
// the last level, whose butterfly is d0 a +- d1 b.  Codes go through a table of value pairs by byte, 16 copies of 8 bytes.
// Bound by HBM and, on TQ4 rows, close to it by the shared-memory pipe (24 wavefronts a row).
#include "tq4_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

namespace w34 {

constexpr int kReadWarps = 8;
constexpr int kReadTableBytes = 256 * 128;
constexpr int kReadTurnBytes = kReadWarps * 4 * 1024;      // four rows a warp change lanes at once

struct ReadParams {
    warp34_kv_layer_layout layout;
    warp34_attention_batch batch;
    uint16_t* out[2];           // K, V
    long long stride[2];        // elements
    int first, sides;           // 0: K first; how many of the two are read
    int aligned;                // output rows start on 16-byte boundaries
    int rows_aligned;           // BF16 rows do
    long long units;            // sides x kv heads x groups of four tokens
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
__device__ __forceinline__ void read_store8(uint16_t* dst, int aligned, const uint32_t (&w)[4]) {
    if (aligned) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { dst[2 * i] = (uint16_t)w[i]; dst[2 * i + 1] = (uint16_t)(w[i] >> 16); }
    }
}

// Place of a 16-byte quad of a row while the columns change lanes: conflict-free for quads stored at 2 (j + 8 (l / 2)) + l % 2 by lane l
// and for the pairs 2 c, 2 c + 1 of chunk c = j + 8 i read by lane j.
__device__ __forceinline__ uint32_t read_quad_place(uint32_t u) { return u ^ ((u >> 3) & 1u) ^ (((u >> 4) & 3u) << 1); }

typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float a, float b) { return (F2)__float_as_uint(a) | ((F2)__float_as_uint(b) << 32); }
__device__ __forceinline__ float f2x(F2 p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float f2y(F2 p) { return __uint_as_float((uint32_t)(p >> 32)); }
__device__ __forceinline__ F2 f2add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 f2mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 f2fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// Butterflies over pair-index bit d of 16 packed pairs.
__device__ __forceinline__ void read_level(F2 (&x)[16], int d, F2 minus_one) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        if (k & d) continue;
        const F2 a = x[k], b = x[k | d];
        x[k] = f2add(a, b);
        x[k | d] = f2fma(b, minus_one, a);
    }
}

// Address of the row of token `tok` (K or V), or 0: the row takes no part.
__device__ __forceinline__ uint64_t read_row_address(const ReadParams& p, int tok, int head, int side) {
    const warp34_attention_batch& b = p.batch;
    if (tok >= b.total_tokens || (b.valid_token_mask != nullptr && b.valid_token_mask[tok] == 0)) return 0;
    const int r = find_request(b.query_start_loc, b.num_reqs, tok);
    if (r < 0 || (b.valid_req_mask != nullptr && b.valid_req_mask[r] == 0)) return 0;
    int page, off;
    if (b.write_slot_mapping != nullptr) {
        const int slot = b.write_slot_mapping[tok];
        if (slot < 0) return 0;
        page = slot >> 4;
        off = slot & 15;
    } else {
        const int q_len = b.query_start_loc[r + 1] - b.query_start_loc[r];
        const int pos = (b.context_lens_before != nullptr ? b.context_lens_before[r] : b.seq_lens_after[r] - q_len) + (tok - b.query_start_loc[r]);
        if (pos < 0 || (pos >> 4) >= b.max_blocks_per_req) return 0;
        page = block_table_page(b.block_tables + (size_t)r * b.max_blocks_per_req, pos >> 4, b.max_blocks_per_req, kInRead);
        off = pos & 15;
    }
    page = pool_page(page, kInRead);
    const warp34_kv_layer_layout& l = p.layout;
    return side == 0 ? l.k_base + (uint64_t)page * l.k_page_stride_bytes + (uint64_t)head * l.k_head_stride_bytes + (uint64_t)off * l.k_token_stride_bytes
                     : l.v_base + (uint64_t)page * l.v_page_stride_bytes + (uint64_t)head * l.v_head_stride_bytes + (uint64_t)off * l.v_token_stride_bytes;
}

// Unit: four tokens of one head, K or V.  Units of a side follow each other by token group, then head.
struct ReadUnit { int tok, head, side; uint64_t row; };
__device__ __forceinline__ ReadUnit read_unit(const ReadParams& p, long long u) {
    ReadUnit x;
    const int heads = p.layout.local_kv_heads;
    const long long g = u / p.sides;
    x.side = p.first + (int)(u - g * p.sides);
    const long long group = g / heads;
    x.head = (int)(g - group * heads);
    x.tok = (int)(4 * group) + (int)((threadIdx.x & 31) >> 3);
    x.row = read_row_address(p, x.tok, x.head, x.side);
    return x;
}

template <bool BF16>
__global__ void __launch_bounds__(kReadWarps * 32, 3) kv_read_tq4_kernel(const ReadParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, j = lane & 7, r4 = lane >> 3;
    for (int i = threadIdx.x; i < 256 * 16; i += kReadWarps * 32) {
        const int byte = i >> 4;
        *reinterpret_cast<float2*>(smem + byte * 128 + (i & 15) * 8) = make_float2(tq4_centroid(byte & 15), tq4_centroid(byte >> 4));
    }
    // signs of this lane's output columns 8 (j + 8 i) + e as sign bits of packed pairs
    uint32_t sign[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = 8 * (j + 8 * i);
        const uint32_t m = c_sign_mask[c >> 5] >> (c & 31);
#pragma unroll
        for (int k = 0; k < 4; ++k) sign[4 * i + k] = (((m >> (2 * k)) & 1u) << 15) | (((m >> (2 * k + 1)) & 1u) << 31);
    }
    grid_dependency_wait();      // nothing above touches global memory
    grid_launch_dependents();
    __syncthreads();
    const uint8_t* table = smem + 8 * (lane & 15);
    uint8_t* turn = smem + kReadTableBytes + (wid * 4 + r4) * 1024;
    const F2 minus_one = f2(-1.0f, -1.0f);
#pragma unroll 1
    for (long long u = (long long)blockIdx.x * kReadWarps + wid; u < p.units; u += (long long)gridDim.x * kReadWarps) {
        const ReadUnit x = read_unit(p, u);
        const uint8_t* row = reinterpret_cast<const uint8_t*>((uintptr_t)x.row);
        F2 v[16];
        float d0 = 0.0f, d1 = 0.0f;
        if (x.row != 0) {
            // quads: register pairs 2 k, 2 k + 1 are columns 8 (k + 8 (j / 2)) + 4 (j % 2) .. + 3
            const uint8_t* codes = row + kTq4BlockBytes * (j >> 2) + 2 + 32 * ((j >> 1) & 1) + 2 * (j & 1);
            uint32_t c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] = *reinterpret_cast<const uint16_t*>(codes + 4 * k);
            d0 = __half2float(*reinterpret_cast<const __half*>(row)) * 0.0625f;
            d1 = __half2float(*reinterpret_cast<const __half*>(row + kTq4BlockBytes)) * 0.0625f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[2 * k] = *reinterpret_cast<const F2*>(table + ((c[k] & 0xffu) << 7));
                v[2 * k + 1] = *reinterpret_cast<const F2*>(table + ((c[k] >> 1) & 0x7f80u));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = 0ull;
        }
        // column bits 0 (inside a pair), 1, 3, 4, 5
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = f2(f2x(v[k]) + f2y(v[k]), f2x(v[k]) - f2y(v[k]));
        read_level(v, 1, minus_one);
        read_level(v, 2, minus_one);
        read_level(v, 4, minus_one);
        read_level(v, 8, minus_one);
        __syncwarp();      // the rows of the unit before have been read
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            *reinterpret_cast<ulonglong2*>(turn + 16 * read_quad_place(2 * (k + 8 * (j >> 1)) + (j & 1))) = make_ulonglong2(v[2 * k], v[2 * k + 1]);
        }
        __syncwarp();
        // chunks: pairs 4 i .. 4 i + 3 are columns 8 (j + 8 i) .. + 7
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(turn + 16 * read_quad_place(2 * (j + 8 * (k >> 1)) + (k & 1)));
            v[2 * k] = q.x;
            v[2 * k + 1] = q.y;
        }
        read_level(v, 2, minus_one);      // column bit 2
        read_level(v, 4, minus_one);      // column bit 6
        const F2 s0 = f2(d0, d0), s1 = f2(d1, d1), n1 = f2(-d1, -d1);
#pragma unroll
        for (int k = 0; k < 8; ++k) {     // column bit 7, and the scales of the two halves
            const F2 a = f2mul(v[k], s0), b = v[k + 8];
            v[k] = f2fma(b, s1, a);
            v[k + 8] = f2fma(b, n1, a);
        }
        if (x.row == 0) continue;
        uint16_t* dst = p.out[x.side] + (size_t)x.tok * (size_t)p.stride[x.side] + (size_t)x.head * kHeadDim + 8 * j;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = read_narrow<BF16>(f2x(v[4 * i + k]), f2y(v[4 * i + k])) ^ sign[4 * i + k];
            read_store8(dst + 64 * i, p.aligned, w);
        }
    }
}

// Rows that are not rotated.  Lane j of a row: chunks j + 8 i.
template <bool BF16>
__global__ void __launch_bounds__(kReadWarps * 32) kv_read_plain_kernel(const ReadParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, j = lane & 7;
#pragma unroll 1
    for (long long u = (long long)blockIdx.x * kReadWarps + wid; u < p.units; u += (long long)gridDim.x * kReadWarps) {
        const ReadUnit x = read_unit(p, u);
        if (x.row == 0) continue;
        const uint8_t* row = reinterpret_cast<const uint8_t*>((uintptr_t)x.row);
        const int format = x.side == 0 ? p.layout.k_format : p.layout.v_format;
        uint32_t raw[4][4];
        float d[4];
        if (format == WARP34_KV_FORMAT_FP8_E4M3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t* src = reinterpret_cast<const uint32_t*>(row + 8 * (j + 8 * i));
                raw[i][0] = src[0];
                raw[i][1] = src[1];
                d[i] = *reinterpret_cast<const float*>(row + kHeadDim + 4 * (i >> 1));
            }
        } else if (format == WARP34_KV_FORMAT_Q8_0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t* src = reinterpret_cast<const uint32_t*>(row + 68 * i + 4 + 8 * j);
                raw[i][0] = src[0];
                raw[i][1] = src[1];
                d[i] = *reinterpret_cast<const float*>(row + 68 * i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t* src = reinterpret_cast<const uint16_t*>(row) + 8 * (j + 8 * i);
                if (p.rows_aligned) {
                    const uint4 q = *reinterpret_cast<const uint4*>(src);
                    raw[i][0] = q.x; raw[i][1] = q.y; raw[i][2] = q.z; raw[i][3] = q.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) raw[i][k] = (uint32_t)src[2 * k] | ((uint32_t)src[2 * k + 1] << 16);
                }
            }
        }
        uint16_t* dst = p.out[x.side] + (size_t)x.tok * (size_t)p.stride[x.side] + (size_t)x.head * kHeadDim + 8 * j;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
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
            read_store8(dst + 64 * i, p.aligned, w);
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
    p.units = (((long long)batch->total_tokens + 3) / 4) * l.local_kv_heads * p.sides;
    const long long needed = (p.units + kReadWarps - 1) / kReadWarps;
    const long long resident = (long long)read_sm_count() * (tq4 ? 3 : 6);
    const unsigned blocks = (unsigned)(needed < resident ? needed : resident);
    cudaStream_t st = (cudaStream_t)ex->stream;
    if (!tq4) return launch_behind(kv_read_plain_kernel<BF16>, dim3(blocks), kReadWarps * 32, 0, st, p);
    const int rc = (int)cudaFuncSetAttribute(kv_read_tq4_kernel<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kReadTableBytes + kReadTurnBytes);
    if (rc != 0) return rc;
    return launch_behind(kv_read_tq4_kernel<BF16>, dim3(blocks), kReadWarps * 32, kReadTableBytes + kReadTurnBytes, st, p);
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
