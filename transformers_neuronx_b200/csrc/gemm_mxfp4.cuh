// What the products with a 4-bit matrix share (gemm_mxfp4.cu: few tokens, gemm_mxfp4_tiles.cu: many).
#pragma once
#include "mxfp4.cuh"
#include "tc_common.cuh"

namespace {

constexpr int TILE_W = 128;                  // rows of W a tile: the accumulator's lanes
constexpr int KB = 64;                       // columns of K in a block of 16-bit values, 128 bytes a row: stages hold two such blocks or a box's four
constexpr int CODE_K = 256;                  // columns of K a box of codes holds: 128 bytes a row
constexpr int CODE_BYTES = TILE_W * CODE_K / 2;

struct Epilogue {
    const float* bias;
    const float* residual;                   // [M, ldc], may be the output
    void* out;
    long long ldc;
    int M, N, act, out_h16, gated;           // N: features of the result
    int vec;                                 // rows of the output, residual and bias allow accesses of four features
};

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// How many of the next stages (up to four) are ready: lane j looks at stage j of one ring, lane 4 + j at stage j of the other, all in one trip
// to shared memory.  A look at a barrier queues behind the MMAs issued before it and takes 150 to 250 cycles even when the stage is ready: a
// look at both rings for every stage left the tensor cores idle for half of the time.
__device__ __forceinline__ int ready_stages(uint64_t* a, int a_slot, uint32_t a_pass, int a_stages, uint64_t* b, int b_slot, uint32_t b_pass, int b_stages) {
    const int lane = threadIdx.x & 31;
    const bool second = lane & 4;
    int s = (second ? b_slot : a_slot) + (lane & 3);
    uint32_t parity = second ? b_pass : a_pass;
    const int n = second ? b_stages : a_stages;
    if (s >= n) { s -= n; parity ^= 1u; }
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32((second ? b : a) + s)), "r"(parity) : "memory");
    const uint32_t ready = __ballot_sync(0xffffffffu, ok);
    __syncwarp();
    return __ffs(~(ready & (ready >> 4) & 15u)) - 1;
}
// D (+)= A B with A read from tensor memory (lane = row, a column = two consecutive values of K).
__device__ __forceinline__ void umma_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__host__ __device__ constexpr uint32_t idesc16(int n) {
    return (1u << 4) | IDESC_H16_AB | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE_W >> 4) << 24);
}

// Activations of results that are rounded to 16 bits anyway (32-bit ones take mx_activation): x / (1 + e^-u) by the same few instructions for silu (u = x)
// and the tanh form of gelu, whose exponential is within 2 + 1.2 |u| units of its last place.  The division gives zero by a divisor of 2^126 and more (u
// below -87.3), an infinity among them, and NaN for an infinity by one, so that nothing has to be held in a range: with e^-u held at e^80, -1e38 became
// -1,800.
__device__ __forceinline__ float gate_fast(float x, float u) { return __fdividef(x, 1.f + __expf(-u)); }
__device__ __forceinline__ float activate(float v, int act) {
    if (act == TNX_ACT_SILU) return gate_fast(v, v);
    if (act == TNX_ACT_GELU_NEW) return gate_fast(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
    return mx_activation(v, act);
}

__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// D = f32, A = B = e2m1, scales 2^(E - 127), both operands K-major, M = 128, N = n; `id`: which half of a column's four scales (0 or 2).
__host__ __device__ constexpr uint32_t idesc4(int n, uint32_t id) {
    return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(TILE_W >> 7) << 27) | (id << 29);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// Eight bytes from any address: aligned words and a shift; [begin, end): the tensor, outside of which nothing is read; `n`: how many bytes are wanted
// (the rest is zero).
__device__ __forceinline__ uint2 load8(const uint8_t* p, const uint8_t* begin, const uint8_t* end, int n) {
    if (n <= 0) return make_uint2(0u, 0u);
    const uint32_t off = (uint32_t)((uintptr_t)p & 3u);
    uint32_t v0, v1;
    if (n >= 8 && off == 0 && ((uintptr_t)p & 7u) == 0) return __ldg((const uint2*)p);
    if (n >= 8 && p - off >= begin && p - off + 12 <= end) {
        const uint32_t* q = (const uint32_t*)(p - off);
        const uint32_t a = __ldg(q), b = __ldg(q + 1), c = off ? __ldg(q + 2) : 0u;
        v0 = __funnelshift_r(a, b, 8 * off); v1 = __funnelshift_r(b, c, 8 * off);
    } else {
        v0 = v1 = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) { const uint32_t E = (uint32_t)__ldg(p + j) << (8 * (j & 3)); if (j < 4) v0 |= E; else v1 |= E; }
    }
    return make_uint2(v0, v1);
}

// ---- host: tensor maps -----------------------------------------------------------------------------
// A [rows, bytes] matrix of bytes in boxes of box_rows x 128 bytes, 128-byte swizzle; and one of 16-bit values in boxes of box_rows x 64.
bool map_bytes(CUtensorMap* out, const void* ptr, int rows, int bytes, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)bytes};
    cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool map_h16(CUtensorMap* out, const void* ptr, int rows, int cols, long long ld, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)KB, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(out, TNX_TMA_H16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline void fill_epilogue(Epilogue& e, const float* bias, const float* residual, void* out, int out_h16, long long ldc, int M, int N, int act, int gated) {
    e.bias = bias; e.residual = residual; e.out = out; e.ldc = ldc;
    e.M = M; e.N = N; e.act = act; e.out_h16 = out_h16; e.gated = gated;
    e.vec = ldc % 4 == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)residual & 15) == 0;
}

}  // namespace
