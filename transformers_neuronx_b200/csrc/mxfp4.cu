// Rows to microscaled 4 bits and back, and the product for sizes that no tensor map can address.  Formats: mxfp4.cuh.
#include "mxfp4.cuh"

namespace {

__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The bits of the largest magnitude of eight values, as a 32-bit float's.  Bits compared as whole numbers put infinities and NaN above every finite value, so
// one comparison finds them.  16-bit values are compared two at a time; four neighbouring lanes hold a block.
__device__ __forceinline__ uint32_t block_max(const Vec8<float>& q) {
    float v[8];
    q.get(v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ uint32_t block_max(const Vec8<h16>& q) {
    const uint32_t s = 0x7FFF7FFFu;
    uint32_t m = __vmaxu2(__vmaxu2(q.raw.x & s, q.raw.y & s), __vmaxu2(q.raw.z & s, q.raw.w & s));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max(m & 0xFFFFu, m >> 16);
#ifdef TNX_F16
    return __float_as_uint(h16_to_float(__ushort_as_half((unsigned short)m)));
#else
    return m << 16;
#endif
}

// Eight values times 2^-e, exactly (or far below the smallest code).
__device__ __forceinline__ void scaled(const Vec8<float>& q, float by, float (&s)[8]) {
    q.get(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= by;
}
__device__ __forceinline__ void scaled(const Vec8<h16>& q, float by, float (&s)[8]) {
#ifdef TNX_F16
    q.get(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= by;
#else
    // bfloat16 halves as operands of a 32-bit multiply-add: nothing to unpack; -0 added leaves the sign of a zero alone
    const uint32_t w[4] = {q.raw.x, q.raw.y, q.raw.z, q.raw.w};
    const unsigned short b = (unsigned short)(__float_as_uint(by) >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("{\n\t.reg .b16 l, h;\n\t"
            "mov.b32 {l, h}, %2;\n\t"
            "fma.rn.f32.bf16 %0, l, %3, %4;\n\t"
            "fma.rn.f32.bf16 %1, h, %3, %4;\n\t}"
            : "=f"(s[2 * i]), "=f"(s[2 * i + 1]) : "r"(w[i]), "h"(b), "f"(-0.f));
#endif
}

// The block's exponent is the smallest e with max |x| <= 6 * 2^e, read off the largest value's bits: m = 1.f * 2^x needs e = x - 2 up to f = 1.5 and
// x - 1 beyond.  The conversion of x * 2^-e rounds to the nearest code, ties to even.
template <typename T>
__device__ __forceinline__ uint32_t quantize8(const Vec8<T>& q, uint32_t& E) {
    const uint32_t m = block_max(q);
    const int e = (int)(m >> 23) - 2 + ((m & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    if (m >= 0x7F800000u) { E = 255u; return 0u; }
    E = (uint32_t)max(e, 0);
    float s[8];
    scaled(q, __uint_as_float((254u - E) << 23), s);              // E <= 253 for finite values
    return pack_e2m1x8(s);
}

// Rows to 4 bits: one read of the values, one write of codes and scales; bound by memory.  `items` = rows * blocks * 4 pieces of eight values, whose
// codes lie in their order.  FLAT: so do the values (whole blocks, no gap between rows, 16-byte aligned), and a thread asks for several pieces
// before it uses the first.  Otherwise a piece's row and column are worked out, and values are read one by one where 16 bytes at a time cannot be.
// 16,384 x 4,096 from bfloat16 29 us, 5.8 TB/s, from 32 bits 45, 6.7 TB/s of which the second-level cache keeps some (bfloat16 with one piece a thread
// 32, three 32, four 37; with each value unpacked and compared alone, four pieces 42); back to bfloat16 28, to 32 bits 65 (two pieces 31 and 65,
// four 28 and 70; 8 blocks an SM that walk 30 and 77).
constexpr int TO_PIECES = 2, TO_BLOCKS = 16, BACK_PIECES = 3, BACK_BLOCKS = 128;          // pieces a thread, blocks an SM at most

// The row of piece i and its first column.
__device__ __forceinline__ long long piece_row(long long i, long long items, int blocks, int& k) {
    const long long row = items <= 0xFFFFFFFFll ? (long long)((unsigned)i / (4u * blocks)) : i / (4 * blocks);
    k = (int)(i - row * (4 * blocks)) * 8;
    return row;
}

template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, long long ld, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                       long long items, int blocks, int K, int vec) {
    pdl_launch_dependents();             // the products read codes behind their own wait
    pdl_wait();
    const long long stride = (long long)gridDim.x * blockDim.x;
    constexpr int U = FLAT ? TO_PIECES : 1;
    // whole warps walk the loop: the block's largest value is found by lanes together
    for (long long i0 = (long long)blockIdx.x * blockDim.x + (threadIdx.x & ~31u); i0 < items; i0 += stride * U) {
        const long long i = i0 + (threadIdx.x & 31u);
        Vec8<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u].zero();
        if (FLAT) {
#pragma unroll
            for (int u = 0; u < U; ++u) if (i + u * stride < items) q[u].load(x + (i + u * stride) * 8);
        } else if (i < items) {
            int k;
            const long long row = piece_row(i, items, blocks, k);
            const T* src = x + row * ld + k;
            if (vec && k + 8 <= K) q[0].load(src);
            else {
                T v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = k + j < K ? src[j] : from_float<T>(0.f);
                memcpy(&q[0], v, sizeof v);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long at = i + u * stride;
            uint32_t E;
            const uint32_t c = quantize8(q[u], E);
            if (at < items) {
                codes[at] = c;
                if ((at & 3) == 0) scales[at >> 2] = (uint8_t)E;
            }
        }
    }
}

// Eight codes as 32-bit numbers, without a scale.
__device__ __forceinline__ void codes_to_float(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    codes_to_f16(w, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*(const __half2*)&h[j]);
        v[2 * j] = f.x; v[2 * j + 1] = f.y;
    }
}

template <typename T>
__device__ __forceinline__ void piece_values(uint32_t c, uint32_t E, Vec8<T>& q) {
    float v[8];
    codes_to_float(c, v);
    const float s = mx_scale(E);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= s;
    q.set(v);
}

// Eight values a thread; bound by memory.  In 32 bits and in bfloat16 every value is exact; float16 rounds what lies outside its range.  No kernel
// behind it starts early: a product may take the values for a matrix that no kernel writes.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, long long ld,
                                                         long long items, int blocks, int K, int vec) {
    pdl_wait();
    const long long stride = (long long)gridDim.x * blockDim.x;
    if (FLAT) {
        constexpr int U = BACK_PIECES;
        for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < items; i += stride * U) {
            uint32_t c[U], E[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long at = i + u * stride;
                c[u] = E[u] = 0u;
                if (at < items) { c[u] = __ldg(codes + at); E[u] = __ldg(scales + (at >> 2)); }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long at = i + u * stride;
                if (at >= items) break;
                Vec8<T> q;
                piece_values(c[u], E[u], q);
                q.store(out + at * 8);
            }
        }
        return;
    }
    // Rows that do not begin on 16 bytes: a warp's 256 values go through shared memory, so that its lanes write neighbouring ones (16,384 x 4,090: 177 us
    // when every lane wrote its eight one by one).
    __shared__ __align__(16) T staged[8][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (long long i0 = (long long)blockIdx.x * blockDim.x + (threadIdx.x & ~31u); i0 < items; i0 += stride) {
        const long long i = i0 + lane < items ? i0 + lane : items - 1;
        int k;
        const long long row = piece_row(i, items, blocks, k), o = row * ld + k;
        const int n = i0 + lane < items ? min(K - k, 8) : 0;
        Vec8<T> q;
        piece_values(__ldg(codes + i), __ldg(scales + (i >> 2)), q);
        if (vec && n == 8) q.store(out + o);
        const unsigned rest = __ballot_sync(0xffffffffu, !(vec && n == 8) && n > 0);
        if (rest == 0u) continue;
        q.store(&staged[warp][lane * 8]);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int from = j * 4 + (lane >> 3), e = lane & 7;
            const long long at = __shfl_sync(0xffffffffu, o, from);
            const int m = __shfl_sync(0xffffffffu, n, from);
            if ((rest >> from & 1u) && e < m) out[at + e] = staged[warp][j * 32 + lane];
        }
        __syncwarp();
    }
}

// The product on the multiply-add units, any sizes, pitches and alignments: a warp per feature (gated: per pair of them) and eight tokens,
// its lanes walk K in pieces of eight codes, 32-bit sums, one order for every number of tokens.
constexpr int SIMT_TOKENS = 8, SIMT_WARPS = 4;
struct SimtParams {
    const void* a; long long lda; int a_kind;              // 0: h16, 1: float, 2: codes (lda then counts blocks)
    const uint8_t* a_scales;
    const uint8_t* codes; const uint8_t* scales;
    const float* bias; const float* residual; void* out; long long ldc;
    int M, N, K, blocks, act, gated, out_h16;               // N: features of the result; gated: the up rows begin at row N
};

__device__ __forceinline__ uint32_t load_codes(const uint8_t* p) {
    return ((uintptr_t)p & 3) == 0 ? *(const uint32_t*)p : (uint32_t)p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16 | (uint32_t)p[3] << 24;
}

__global__ void __launch_bounds__(32 * SIMT_WARPS) simt_kernel(const SimtParams p) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int n = blockIdx.x * SIMT_WARPS + (threadIdx.x >> 5);
    const int m0 = blockIdx.y * SIMT_TOKENS;
    if (n >= p.N) return;
    float sum[2][SIMT_TOKENS];
#pragma unroll
    for (int t = 0; t < SIMT_TOKENS; ++t) sum[0][t] = sum[1][t] = 0.f;
    for (int piece = lane; piece < p.blocks * 4; piece += 32) {
        const int k = piece * 8;
        float w[2][8];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (g && !p.gated) break;
            const long long row = n + (long long)g * p.N;
            const uint32_t c = load_codes(p.codes + row * p.blocks * 16 + piece * 4);
            const float s = mx_scale(p.scales[row * p.blocks + (piece >> 2)]);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[g][j] = mx_code(c >> (4 * j)) * s;
        }
#pragma unroll
        for (int t = 0; t < SIMT_TOKENS; ++t) {
            if (m0 + t >= p.M) break;
            const long long row = m0 + t;
            float x[8];
            if (p.a_kind == 2) {
                const uint32_t c = load_codes((const uint8_t*)p.a + row * p.blocks * 16 + piece * 4);
                const float s = mx_scale(p.a_scales[row * p.blocks + (piece >> 2)]);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = mx_code(c >> (4 * j)) * s;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = k + j >= p.K ? 0.f : p.a_kind ? ((const float*)p.a)[row * p.lda + k + j] : h16_to_float(((const h16*)p.a)[row * p.lda + k + j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum[0][t] = fmaf(w[0][j], x[j], sum[0][t]);
                if (p.gated) sum[1][t] = fmaf(w[1][j], x[j], sum[1][t]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < SIMT_TOKENS; ++t) {
        if (m0 + t >= p.M) break;
        float v = warp_sum(sum[0][t]), u = p.gated ? warp_sum(sum[1][t]) : 0.f;
        if (lane == 0) {
            if (p.bias) { v += p.bias[n]; if (p.gated) u += p.bias[p.N + n]; }
            v = mx_activation(v, p.act);
            if (p.gated) v *= u;
            const long long o = (long long)(m0 + t) * p.ldc + n;
            if (p.residual) v += p.residual[o];
            if (p.out_h16) ((h16*)p.out)[o] = float_to_h16(v);
            else ((float*)p.out)[o] = v;
        }
    }
}

// Blocks of 256 threads, `most` an SM at most.
inline unsigned grid_for(long long items, int pieces, int most, int sms) {
    const long long want = (items + 256 * pieces - 1) / (256 * pieces), limit = (long long)sms * most;
    return (unsigned)(want < limit ? want : limit);
}

template <typename T>
int launch_quantize(const void* x, long long ld, void* codes, void* scales, int rows, int K, int sms, cudaStream_t stream) {
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    const long long items = (long long)rows * blocks * 4;
    const int vec = ld % 8 == 0 && ((uintptr_t)x & 15) == 0;
    // a few rows: a piece a thread, so that all SMs have some
    if (vec && K % MX_BLOCK == 0 && (ld == K || rows == 1))
        return tnx_launch_ex(1, quantize_kernel<T, true>, dim3(grid_for(items, items > 256ll * 8 * sms ? TO_PIECES : 1, TO_BLOCKS, sms)), dim3(256), 0, stream, (const T*)x, ld,
                             (uint32_t*)codes, (uint8_t*)scales, items, blocks, K, vec);
    return tnx_launch_ex(1, quantize_kernel<T, false>, dim3(grid_for(items, 1, TO_BLOCKS, sms)), dim3(256), 0, stream, (const T*)x, ld, (uint32_t*)codes,
                         (uint8_t*)scales, items, blocks, K, vec);
}

template <typename T>
int launch_dequantize(const void* codes, const void* scales, void* out, long long ld, int rows, int K, int sms, cudaStream_t stream) {
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    const long long items = (long long)rows * blocks * 4;
    const int vec = ld % 8 == 0 && ((uintptr_t)out & 15) == 0;
    if (vec && K % MX_BLOCK == 0 && (ld == K || rows == 1))
        return tnx_launch_ex(1, dequantize_kernel<T, true>, dim3(grid_for(items, items > 256ll * 8 * sms ? BACK_PIECES : 1, BACK_BLOCKS, sms)), dim3(256), 0, stream,
                             (const uint32_t*)codes, (const uint8_t*)scales, (T*)out, ld, items, blocks, K, vec);
    return tnx_launch_ex(1, dequantize_kernel<T, false>, dim3(grid_for(items, 1, BACK_BLOCKS, sms)), dim3(256), 0, stream, (const uint32_t*)codes, (const uint8_t*)scales,
                         (T*)out, ld, items, blocks, K, vec);
}

}  // namespace

// x: [rows, K] of the 16-bit type or float, row pitch ld elements; codes 4-byte aligned.
TNX_EXPORT int tnx_mxfp4_quantize(const void* x, int x_h16, long long ld, void* codes, void* scales, int rows, int K, int sms, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (K <= 0 || sms <= 0 || ((uintptr_t)codes & 3)) return TNX_ERR_BAD_ARG;
    return x_h16 ? launch_quantize<h16>(x, ld, codes, scales, rows, K, sms, stream) : launch_quantize<float>(x, ld, codes, scales, rows, K, sms, stream);
}

TNX_EXPORT int tnx_mxfp4_dequantize(const void* codes, const void* scales, void* out, int out_h16, long long ld, int rows, int K, int sms, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (K <= 0 || sms <= 0 || ((uintptr_t)codes & 3)) return TNX_ERR_BAD_ARG;
    return out_h16 ? launch_dequantize<h16>(codes, scales, out, ld, rows, K, sms, stream) : launch_dequantize<float>(codes, scales, out, ld, rows, K, sms, stream);
}

TNX_EXPORT int tnx_mxfp4_gemm_simt(const void* a, int a_kind, const void* a_scales, long long lda, const void* codes, const void* scales, const float* bias,
                                   const float* residual, void* out, int out_h16, long long ldc, int M, int N, int K, int act, int gated, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || a_kind < 0 || a_kind > 2 || act < 0 || act >= TNX_ACT_COUNT) return TNX_ERR_BAD_ARG;
    SimtParams p;
    p.a = a; p.lda = lda; p.a_kind = a_kind; p.a_scales = (const uint8_t*)a_scales;
    p.codes = (const uint8_t*)codes; p.scales = (const uint8_t*)scales;
    p.bias = bias; p.residual = residual; p.out = out; p.ldc = ldc;
    p.M = M; p.N = N; p.K = K; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK; p.act = act; p.gated = gated; p.out_h16 = out_h16;
    // 65,535 blocks along y at most: more tokens go in slices
    const int slice = 65535 * SIMT_TOKENS;
    for (long long m = 0; m < M; m += slice) {            // (an int would pass its end behind the last slice of nearly 2^31 tokens)
        SimtParams q = p;
        q.M = M - m < slice ? (int)(M - m) : slice;
        q.a = a_kind == 2 ? (const void*)((const uint8_t*)a + m * p.blocks * 16) : (const void*)((const char*)a + m * lda * (a_kind ? 4 : 2));
        if (a_scales) q.a_scales = p.a_scales + m * p.blocks;
        if (residual) q.residual = residual + m * ldc;
        q.out = (char*)out + m * ldc * (out_h16 ? 2 : 4);
        const int r = tnx_launch_ex(1, simt_kernel, dim3((N + SIMT_WARPS - 1) / SIMT_WARPS, (q.M + SIMT_TOKENS - 1) / SIMT_TOKENS), dim3(32 * SIMT_WARPS), 0, stream, q);
        if (r) return r;
    }
    return 0;
}

// The same with the parameters in one array (the stream last): a call through ctypes costs 0.1 us a parameter.
TNX_EXPORT int tnx_mxfp4_quantize_packed(const long long* v) {
    return tnx_mxfp4_quantize((const void*)v[0], (int)v[1], (long long)v[2], (void*)v[3], (void*)v[4], (int)v[5], (int)v[6], (int)v[7], (cudaStream_t)v[8]);
}
TNX_EXPORT int tnx_mxfp4_dequantize_packed(const long long* v) {
    return tnx_mxfp4_dequantize((const void*)v[0], (const void*)v[1], (void*)v[2], (int)v[3], (long long)v[4], (int)v[5], (int)v[6], (int)v[7], (cudaStream_t)v[8]);
}
TNX_EXPORT int tnx_mxfp4_gemm_simt_packed(const long long* v) {
    return tnx_mxfp4_gemm_simt((const void*)v[0], (int)v[1], (const void*)v[2], (long long)v[3], (const void*)v[4], (const void*)v[5],
                               (const float*)v[6], (const float*)v[7], (void*)v[8], (int)v[9], (long long)v[10], (int)v[11], (int)v[12], (int)v[13],
                               (int)v[14], (int)v[15], (cudaStream_t)v[16]);
}
