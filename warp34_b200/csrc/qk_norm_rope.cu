// Norm and rotary embedding of every query and key head, and the split of the layer's output gate, in one pass over packed
// projection rows:
//
//   y = x * rsqrt(mean(x^2) + eps) * (weight_offset + w)          per head row of 256, fp32
//   y[i], y[i + h] <- y[i] cos a_i - y[i + h] sin a_i, y[i + h] cos a_i + y[i] sin a_i      for i < h = rotary_dim / 2
//   a_i = position * inv_freq[i]
//
// and one rounding to the activation type at the end.  (The producer in front of the TQ4 append, tq4_append.cu, is the
// reference's K half with its two roundings, and appends what it makes; this one is for every layer format and the query half.)
//
// A head row is a warp: 8 columns a lane, one 16-byte access each way.  Angles: the frequency becomes turns per position as a
// 64-bit fraction, whose product with the position wraps modulo one turn by itself; what is left is off by 2^-32 turns, 2^-52 of the
// whole angle and, as a float of up to half a turn, 2^-26 turns = 1e-7 rad (a product in fp32 is off by 2^-7 rad at position 131072).  Sine and cosine are made once per token and block
// (sincospif) and shared by its heads through shared memory, while the rows are on their way.
//
// Bound by HBM: on 32768 tokens of 24 query heads with gate and 4 key heads (1745 MB) the kernel takes 268 us, the measured copy rate, and a
// call among others on changing inputs 295, 0.92 of it; without a gate (940 MB) the kernel takes 221 us, 0.66 of it, half of the issue slots taken.
#include "tq4_common.cuh"

#include <cuda_bf16.h>

namespace w34 {

constexpr int kQkWarps = 8;
constexpr int kQkBlocks = 4;      // of eight warps an SM: registers of 32 rows of loads in flight

struct QkParams {
    warp34_qk_norm_rope_args a;
    int rows;         // query and key heads of a token
    int aligned;      // every row starts on a 16-byte boundary
};

__device__ __forceinline__ void qk_load8(const uint16_t* src, int aligned, uint32_t (&w)[4]) {
    if (aligned) {
        const uint4 q = *reinterpret_cast<const uint4*>(src);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16);
    }
}
__device__ __forceinline__ void qk_store8(uint16_t* dst, int aligned, const uint32_t (&w)[4]) {
    if (aligned) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { dst[2 * i] = (uint16_t)w[i]; dst[2 * i + 1] = (uint16_t)(w[i] >> 16); }
    }
}
template <bool BF16>
__device__ __forceinline__ float2 qk_widen(uint32_t w) {
    return BF16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t qk_narrow(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Frequency in radians per position -> turns per position modulo 1, as a 64-bit fraction.
__device__ __forceinline__ unsigned long long turns_of(float inv_freq) {
    const double x = (double)inv_freq * 0.15915494309189533577;      // 1 / (2 pi)
    return __double2ull_rz((x - floor(x)) * 18446744073709551616.0);
}

// Block: one token, (warps of the block) * ROWS of its head rows (blockIdx.y counts them).
template <bool BF16, int ROWS, bool GATED>
__global__ void __launch_bounds__(kQkWarps * 32, kQkBlocks) qk_norm_rope_kernel(const QkParams p) {
    __shared__ __align__(16) float s_cos[kHeadDim / 2], s_sin[kHeadDim / 2];
    grid_dependency_wait();
    grid_launch_dependents();
    const warp34_qk_norm_rope_args& a = p.a;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const size_t tok = blockIdx.x;
    if (a.valid_token_mask != nullptr && a.valid_token_mask[tok] == 0) return;      // block-uniform
    const int warps = (int)(blockDim.x >> 5), row0 = (int)blockIdx.y * (warps * ROWS) + wid;
    constexpr int q_width = GATED ? 2 * kHeadDim : kHeadDim;

    uint32_t x[ROWS][4], gate[GATED ? ROWS : 1][4];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + warps * i;
        if (row < a.num_q_heads) {
            const uint16_t* src = static_cast<const uint16_t*>(a.q_in) + tok * (size_t)a.q_in_stride + (size_t)row * q_width + 8 * lane;
            qk_load8(src, p.aligned, x[i]);
            if (GATED) qk_load8(src + kHeadDim, p.aligned, gate[GATED ? i : 0]);
        } else if (row < p.rows) {
            qk_load8(static_cast<const uint16_t*>(a.k_in) + tok * (size_t)a.k_in_stride + (size_t)(row - a.num_q_heads) * kHeadDim + 8 * lane, p.aligned, x[i]);
        }
    }
    const int half = a.rotary_dim >> 1;
    for (int i = threadIdx.x; i < half; i += (int)blockDim.x) {
        int plane = 0;
        if (a.position_planes == 3) {
            if (i % 3 == 1 && i < 3 * a.mrope_s1) plane = 1;
            else if (i % 3 == 2 && i < 3 * a.mrope_s2) plane = 2;
        }
        const long long pos = a.positions[(size_t)plane * (size_t)a.position_plane_stride + tok];
        const unsigned long long turn = (unsigned long long)pos * turns_of(a.inv_freq[i]);
        // the fraction of a turn, rounded to 32 bits and read as signed: half turns in [-1, 1)
        const int frac = (int)(uint32_t)((turn + 0x80000000ull) >> 32);
        float sn, cs;
        sincospif((float)frac * 4.656612873077393e-10f, &sn, &cs);
        s_cos[i] = cs;
        s_sin[i] = sn;
    }
    __syncthreads();

    // this lane's part in the rotation: columns below `half` take -sin of their partner
    const int lanes_half = half >> 3;
    const bool rotates = lane < 2 * lanes_half, low = lane < lanes_half;
    const int partner = rotates ? (low ? lane + lanes_half : lane - lanes_half) : lane;
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { cs[e] = 1.0f; sn[e] = 0.0f; }
    if (rotates) {
        const int at = 8 * (low ? lane : lane - lanes_half);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const float4 c = *reinterpret_cast<const float4*>(&s_cos[at + 4 * v]), s = *reinterpret_cast<const float4*>(&s_sin[at + 4 * v]);
            cs[4 * v] = c.x; cs[4 * v + 1] = c.y; cs[4 * v + 2] = c.z; cs[4 * v + 3] = c.w;
            sn[4 * v] = low ? -s.x : s.x; sn[4 * v + 1] = low ? -s.y : s.y; sn[4 * v + 2] = low ? -s.z : s.z; sn[4 * v + 3] = low ? -s.w : s.w;
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + warps * i;
        if (row >= p.rows) break;      // warp-uniform
        const bool is_q = row < a.num_q_heads;
        float v[8], ss = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = qk_widen<BF16>(x[i][k]);
            v[2 * k] = f.x;
            v[2 * k + 1] = f.y;
            ss = __fmaf_rn(f.x, f.x, __fmaf_rn(f.y, f.y, ss));
        }
        ss = warp_sum(ss);
        const float inv = rsqrtf(__fmaf_rn(ss, 1.0f / kHeadDim, a.rms_eps));
        uint32_t w[4];
        qk_load8(static_cast<const uint16_t*>(is_q ? a.q_norm_w : a.k_norm_w) + 8 * lane, p.aligned, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = qk_widen<BF16>(w[k]);
            v[2 * k] *= inv * (a.weight_offset + f.x);
            v[2 * k + 1] *= inv * (a.weight_offset + f.y);
        }
        if (half != 0) {      // block-uniform
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float other = __shfl_sync(0xffffffffu, v[e], partner);
                if (rotates) v[e] = __fmaf_rn(v[e], cs[e], other * sn[e]);
            }
        }
        uint32_t out[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = qk_narrow<BF16>(v[2 * k], v[2 * k + 1]);
        if (is_q) {
            qk_store8(static_cast<uint16_t*>(a.q_out) + tok * (size_t)a.q_out_stride + (size_t)row * kHeadDim + 8 * lane, p.aligned, out);
            if (GATED) qk_store8(static_cast<uint16_t*>(a.gate_out) + tok * (size_t)a.gate_out_stride + (size_t)row * kHeadDim + 8 * lane, p.aligned, gate[GATED ? i : 0]);
        } else {
            qk_store8(static_cast<uint16_t*>(a.k_out) + tok * (size_t)a.k_out_stride + (size_t)(row - a.num_q_heads) * kHeadDim + 8 * lane, p.aligned, out);
        }
    }
}

template <bool BF16>
static int launch_qk_norm_rope(const warp34_exec* ex, const warp34_qk_norm_rope_args* args) {
    if (ex == nullptr || args == nullptr) return (int)cudaErrorInvalidValue;
    const warp34_qk_norm_rope_args& a = *args;
    if (a.num_tokens < 0 || a.num_q_heads < 0 || a.num_kv_heads < 0 || a.rotary_dim < 0) return (int)cudaErrorInvalidValue;
    if (a.head_dim != kHeadDim || a.rotary_dim > kHeadDim || (a.rotary_dim & 15) != 0) return (int)cudaErrorNotSupported;
    const long long q_cols = (long long)a.num_q_heads * kHeadDim, k_cols = (long long)a.num_kv_heads * kHeadDim;
    const bool gated = a.gate_out != nullptr;
    if (a.num_q_heads > 0 && (a.q_in == nullptr || a.q_out == nullptr || a.q_norm_w == nullptr || a.q_in_stride < (gated ? 2 : 1) * q_cols ||
                              a.q_out_stride < q_cols || (gated && a.gate_out_stride < q_cols))) {
        return (int)cudaErrorInvalidValue;
    }
    if (a.num_kv_heads > 0 && (a.k_in == nullptr || a.k_out == nullptr || a.k_norm_w == nullptr || a.k_in_stride < k_cols || a.k_out_stride < k_cols)) {
        return (int)cudaErrorInvalidValue;
    }
    if (a.rotary_dim > 0 && (a.positions == nullptr || a.inv_freq == nullptr || (a.position_planes != 1 && a.position_planes != 3) ||
                             (a.position_planes == 3 && a.position_plane_stride < a.num_tokens))) {
        return (int)cudaErrorInvalidValue;
    }
    QkParams p;
    p.a = a;
    const long long rows = (long long)a.num_q_heads + a.num_kv_heads;
    if (a.num_tokens == 0 || rows == 0) return 0;
    if (rows > 65535) return (int)cudaErrorInvalidValue;
    p.rows = (int)rows;
    uintptr_t odd = 0, bits = 0;      // of used pointers and strides, in bytes
    if (a.num_q_heads > 0) {
        bits |= (uintptr_t)a.q_in | (uintptr_t)a.q_out | (uintptr_t)a.q_norm_w | (uintptr_t)(2 * a.q_in_stride) | (uintptr_t)(2 * a.q_out_stride);
        odd |= (uintptr_t)a.q_in | (uintptr_t)a.q_out | (uintptr_t)a.q_norm_w;
        if (gated) {
            bits |= (uintptr_t)a.gate_out | (uintptr_t)(2 * a.gate_out_stride);
            odd |= (uintptr_t)a.gate_out;
        }
    }
    if (a.num_kv_heads > 0) {
        bits |= (uintptr_t)a.k_in | (uintptr_t)a.k_out | (uintptr_t)a.k_norm_w | (uintptr_t)(2 * a.k_in_stride) | (uintptr_t)(2 * a.k_out_stride);
        odd |= (uintptr_t)a.k_in | (uintptr_t)a.k_out | (uintptr_t)a.k_norm_w;
    }
    if ((odd & 1u) != 0u) return (int)cudaErrorInvalidValue;
    p.aligned = (bits & 15u) == 0u ? 1 : 0;
    cudaStream_t st = (cudaStream_t)ex->stream;
    // Four rows a warp share the token's angles; few tokens take a row a warp, so that more SMs work on each.
    const bool wide = (long long)a.num_tokens * rows >= 148ll * 8 * kQkWarps;
    // As many warps as the token's rows fill: 28 rows take seven.
    const unsigned each = wide ? 4u : 1u, need = ((unsigned)rows + each - 1) / each, blocks = (need + kQkWarps - 1) / kQkWarps;
    const unsigned warps = (need + blocks - 1) / blocks;
    const dim3 grid((unsigned)a.num_tokens, blocks);
    if (gated) {
        return wide ? launch_behind(qk_norm_rope_kernel<BF16, 4, true>, grid, warps * 32, 0, st, p)
                    : launch_behind(qk_norm_rope_kernel<BF16, 1, true>, grid, warps * 32, 0, st, p);
    }
    return wide ? launch_behind(qk_norm_rope_kernel<BF16, 4, false>, grid, warps * 32, 0, st, p)
                : launch_behind(qk_norm_rope_kernel<BF16, 1, false>, grid, warps * 32, 0, st, p);
}

}  // namespace w34

extern "C" int warp34_qk_norm_rope_f16(const warp34_exec* ex, const warp34_qk_norm_rope_args* args) {
    return w34::launch_qk_norm_rope<false>(ex, args);
}
extern "C" int warp34_qk_norm_rope_bf16(const warp34_exec* ex, const warp34_qk_norm_rope_args* args) {
    return w34::launch_qk_norm_rope<true>(ex, args);
}
