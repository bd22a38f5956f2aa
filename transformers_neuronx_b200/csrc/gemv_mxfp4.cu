// Products of a few tokens with a 4-bit matrix (formats: mxfp4.cuh; what is computed: gemm_mxfp4.cu).  The matrix is streamed once; what
// bounds them is memory, or else the instructions that turn codes into operands, so these are few.  One token by 16,384 x 4,096 11 to 12 us,
// 3 TB/s, of which 3.5 are what the smallest call takes (8.3 without scales, activations and arithmetic); eight 13 (float16) and 16 (bfloat16); one by
// 5,120 x 20,480 18 us.
//
// A warp takes 16 rows of W (gated: 8 gate rows and their 8 up rows) and a share of K, which one more warp fetches through TMA in boxes of
// 256 columns, four ahead.  A block of 32 columns is two MMAs (mma.sync m16n8k16, 16 rows by 8
// tokens): which column of K stands where in an MMA is free as long as both operands agree, so a lane multiplies eight neighbouring columns
// of its two rows, one 32-bit word of codes each.  The conversion e2m1x2 -> f16x2 makes them operands, two an instruction and without their
// scale: an MMA's columns belong to one block, so its 32-bit sums are multiplied by the block's scale when they are added up.  (Codes looked
// up in a table of the block's scaled magnitudes by byte permutation took 15 instructions for eight values, which the half-rate unit that
// executes them all bounded: 24 us for one token by 16,384 x 4,096, at 1.5 TB/s.)
//
// Activations are float16 operands too: float16 as they are, others divided by a power of two that brings the largest of a box's 256 to
// 2^14..2^15, in one term (bfloat16's eight bits and 4-bit values fit) or three (32 bits).  What is lost is below 2^-39 of the largest of
// the 256, where float16 ends.  A block's sum of such operands is up to 2^15 times too large when it meets the matrix's scale, so that by scale bytes from
// 228 on it may leave 32 bits where the result does not: a sum that is not finite is worked out again in 64 bits, if its row has such a scale.
// (Choosing another way for them ahead, by a look at the scales, took 4 to 7% of one token by 16,384 x 4,096.)
//
// The warps of a block: wf groups of 16 rows by wk shares of K, whose sums meet in shared memory; K may be split further over the blocks of a
// cluster.  The plan chooses them so that one round of blocks, one an SM, covers the GPU as evenly as the sizes allow.
#include "mxfp4.cuh"
#include "tc_common.cuh"

namespace {

constexpr int MAX_WARPS = 15;               // and one that fetches
constexpr int SLOT_K = 256, SLOT_BLOCKS = SLOT_K / MX_BLOCK, SLOT_BYTES = 16 * SLOT_K / 2;
constexpr int AHEAD = 4;                     // boxes a warp has asked for

struct Params {
    const void* a; const uint8_t* a_scales; long long lda;
    int a_kind, a_vec;                       // 0: h16, 1: float, 2: codes; rows can be read 16 bytes at a time
    const uint8_t* codes; const uint8_t* scales;
    const float* bias; const float* residual; void* out; long long ldc;
    int M, N, K, w_rows, blocks, slots, act, out_h16, gated;
    int wf, wk, splits, slots_per_split, phase; // phase: boxes of K whose activations lie in shared memory at a time
    int x_at, sx_at;                         // places in shared memory
    int sw_at, sw_ld, words;                 // scales' place, bytes a row of them; eight of them are one aligned load
    int* err;
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Shared memory by its own addresses: a pointer made from a rounded-up address is a generic one to the compiler, and 64-bit arithmetic on those and
// generic loads were a third of the main loop's instructions.
__device__ __forceinline__ uint32_t lds32(uint32_t a) { uint32_t v; asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a)); return v; }
__device__ __forceinline__ uint32_t lds16(uint32_t a) { uint16_t v; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a)); return v; }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ float2 lds_f2(uint32_t a) { float2 v; asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a)); return v; }

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *(const uint32_t*)&r;
}

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Eight bytes to shared memory, the first n of them from src, the others zero; cp.async.wait_all waits for them.
__device__ __forceinline__ void copy8_async(void* dst, const void* src, uint32_t n) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void copy16_async(void* dst, const void* src, uint32_t n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}

// Eight activations of a token from column k on, as they lie in memory.
struct Raw { uint4 a, b; };
__device__ __forceinline__ Raw load_raw(const Params& p, int token, int k) {
    Raw r;
    r.a = r.b = make_uint4(0u, 0u, 0u, 0u);
    if (p.a_kind == 2) {
        if (k < p.blocks * MX_BLOCK) {
            const long long b = (long long)token * p.blocks + (k >> 5);
            r.a.x = __ldg((const uint32_t*)((const uint8_t*)p.a + b * 16 + ((k & 31) >> 1)));
            r.a.y = __ldg(p.a_scales + b);
        }
    } else if (p.a_vec && k + 8 <= p.K) {
        const char* at = (const char*)p.a + (token * p.lda + k) * (p.a_kind ? 4 : 2);
        r.a = __ldg((const uint4*)at);
        if (p.a_kind) r.b = __ldg((const uint4*)at + 1);
    } else if (p.a_kind) {
        const float* src = (const float*)p.a + token * p.lda + k;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < p.K ? __ldg(src + j) : 0.f;
        r.a = *(const uint4*)&v[0]; r.b = *(const uint4*)&v[4];
    } else {
        const h16* src = (const h16*)p.a + token * p.lda + k;
        h16 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < p.K ? src[j] : float_to_h16(0.f);
        r.a = *(const uint4*)&v[0];
    }
    return r;
}

// A warp's pieces of eight columns are the 256 of a box.  They become TERMS float16 numbers each whose sum times `scale`, a power of two that
// all 256 share, they are: the largest lies between 2^14 and 2^15.
template <int TERMS, bool SCALED>
__device__ __forceinline__ void make_terms(const Params& p, const Raw& r, uint4 (&out)[TERMS], float& scale) {
    if (!SCALED) { out[0] = r.a; scale = 1.f; return; }
    float v[8];
    if (p.a_kind == 2) {
        const float s = mx_scale(r.a.y);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = mx_code(r.a.x >> (4 * j)) * s;
    } else if (p.a_kind) {
        v[0] = __uint_as_float(r.a.x); v[1] = __uint_as_float(r.a.y); v[2] = __uint_as_float(r.a.z); v[3] = __uint_as_float(r.a.w);
        v[4] = __uint_as_float(r.b.x); v[5] = __uint_as_float(r.b.y); v[6] = __uint_as_float(r.b.z); v[7] = __uint_as_float(r.b.w);
    } else {
        Vec8<h16> q;
        q.raw = r.a;
        q.get(v);
    }
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    m = __reduce_max_sync(0xffffffffu, m);
    const uint32_t f = min(268u - (m >> 23), 254u);                  // 2^(14 - exponent of the largest), a normal number
    const float by = __uint_as_float(f << 23);
    scale = __uint_as_float(f < 254u ? (254u - f) << 23 : 0x00400000u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= by;
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = pack_f16(v[2 * j], v[2 * j + 1]);
            if (t + 1 < TERMS) {
                const float2 h = __half22float2(*(const __half2*)&w[j]);
                // what is not finite is whole in the first term (a rest would be NaN for an infinity)
                v[2 * j] = fabsf(h.x) < INFINITY ? v[2 * j] - h.x : 0.f;
                v[2 * j + 1] = fabsf(h.y) < INFINITY ? v[2 * j + 1] - h.y : 0.f;
            }
        }
        out[t] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A scale byte as a 32-bit number, in the byte's place `at` of w: 2^-127 is half of the smallest normal number; 255, an infinity by its bits,
// becomes NaN.
__device__ __forceinline__ float scale_at(uint32_t w, int at) {
    const float f = __uint_as_float(max((at < 3 ? w << (23 - 8 * at) : w >> 1) & 0x7F800000u, 0x00400000u));
    return fmaf(f, 0.f, f);
}

// sum_k a[k] w[k] by one thread, in 64 bits: a row of codes and its scales, a token's activations (a_scales: of codes).  `v`: the sum as it came out, not
// finite, which is right where no scale is from HIGH_SCALE to 254 (activations or blocks that are not finite).  (Single parameters: the kernel's as a whole
// would be copied to memory of its own at the kernel's start, 2 us.)
constexpr uint32_t HIGH_SCALE = 228u;        // eight blocks' sums, 2^26 at the most, times a smaller scale stay in 32 bits
__device__ __forceinline__ double power_of_two(uint32_t E) { return E == 255u ? (double)NAN : __hiloint2double((int)((E + 896u) << 20), 0); }      // 2^(E - 127)
__device__ __noinline__ float sum_again(float v, const uint8_t* codes, const uint8_t* scales, const void* a, const uint8_t* a_scales, int a_kind, int K) {
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    int b = 0;
    if (((uintptr_t)scales & 3) == 0)                     // four bytes at a time up to the first of HIGH_SCALE or more
        for (; b + 4 <= blocks; b += 4) {
            const uint32_t w = __ldg((const uint32_t*)(scales + b));
            if (((w & 0x7F7F7F7Fu) + 0x01010101u * (256u - HIGH_SCALE)) & w & 0x80808080u) break;
        }
    while (b < blocks && (scales[b] < HIGH_SCALE || scales[b] == 255u)) ++b;
    if (b == blocks) return v;
    double sum = 0.;
#pragma unroll 1
    for (int k = 0; k < K; ++k) {
        float x;
        if (a_kind == 2) x = mx_code(((const uint8_t*)a)[k / 2] >> (4 * (k & 1)));
        else x = a_kind ? ((const float*)a)[k] : h16_to_float(((const h16*)a)[k]);
        const double w = mx_code(codes[k / 2] >> (4 * (k & 1))) * power_of_two(scales[k / MX_BLOCK]);
        sum += w * (a_kind == 2 ? x * power_of_two(a_scales[k / MX_BLOCK]) : (double)x);
    }
    return (float)sum;
}

// NT: groups of eight tokens; SCALED: the activations have scales.  Warps 0 .. wf * wk - 1 multiply, the last one fetches codes.
template <int TERMS, int NT, bool SCALED>
__global__ void __launch_bounds__(32 * (MAX_WARPS + 1), 1) gemv_kernel(const __grid_constant__ CUtensorMap map_w, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[MAX_WARPS][AHEAD], empty[MAX_WARPS][AHEAD];
    const int warps = p.wf * p.wk, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wf = warp % p.wf, wk = warp / p.wf;
    const int s_begin = (int)blockIdx.z * p.slots_per_split, s_end = min(p.slots, s_begin + p.slots_per_split);
    const int per = (s_end - s_begin + p.wk - 1) / p.wk;              // boxes of a share of K
    const int step = p.gated ? 8 : 16, first = blockIdx.x * p.wf * step;             // this block's first feature
    const int box_bytes = p.wf * SLOT_BYTES;                          // a share's boxes: rows first.., then rows second.. of all its warps
    bool ok = true;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.wk; ++i)
            for (int j = 0; j < AHEAD; ++j) { mbar_init(&full[i][j], 1); mbar_init(&empty[i][j], p.wf); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    __syncthreads();
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

    if (warp == warps) {
        if (lane == 0)
            for (int i = 0; i < per && ok; ++i)
                for (int share = 0; share < p.wk && ok; ++share) {
                    const int s = s_begin + share * per + i, place = i % AHEAD;
                    if (s >= s_end) break;
                    if (i >= AHEAD) { ok = mbar_wait(&empty[share][place], (uint32_t)(i / AHEAD - 1) & 1u, p.err, 82); if (!ok) break; }
                    uint8_t* at = smem + (share * AHEAD + place) * box_bytes;
                    mbar_expect_tx(&full[share][place], (uint32_t)box_bytes);
                    tma_load_2d(at, &map_w, &full[share][place], s * (SLOT_K / 2), first);
                    tma_load_2d(at + box_bytes / 2, &map_w, &full[share][place], s * (SLOT_K / 2), p.gated ? p.N + first : first + 8 * p.wf);
                }
        __syncwarp();
    } else {
        const int b = min(s_begin + wk * per, s_end), e = min(b + per, s_end);
        uint4* xs = (uint4*)(smem + p.x_at);              // [term][box of the phase][block][NT * 8 tokens][lane t]; rows of no token are never read out
        float* sx = (float*)(smem + p.sx_at);             // [box of the phase][NT * 8 tokens]
        uint8_t* sw = smem + p.sw_at;                     // [row: the first half's, then the second's][box of the phase][8 scales]
        constexpr int BLOCK_X = NT * 8 * 4, BOX_X = SLOT_BLOCKS * BLOCK_X;
        const int term_step = p.phase * p.wk * BOX_X;
        int place = 0;
        uint32_t pass = 0u;
        // A phase is the next p.phase boxes of every share of K.
        for (int f0 = 0; f0 < per; f0 += p.phase) {
            if (f0) asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory");
            const int len = min(p.phase, per - f0);       // boxes of a share
            // W's scales, as they lie in memory: a trip there for every box would take longer than the box.  Copied without waiting for each: a thread
            // has several, whose trips one after the other took 3 to 4 us.
            for (int q = threadIdx.x; q < 16 * p.wf * p.wk * len; q += 32 * warps) {
                const int row = q / (p.wk * len), rest = q - row * (p.wk * len), share = rest / len, f = rest - share * len;
                const int w_row = min(row < 8 * p.wf ? first + row : (p.gated ? p.N + first : first + 8 * p.wf) + row - 8 * p.wf, p.w_rows - 1);
                const int blk = (s_begin + share * per + f0 + f) * SLOT_BLOCKS;
                const uint8_t* src = p.scales + (long long)w_row * p.blocks + blk;
                uint8_t* to = sw + row * p.sw_ld + (share * p.phase + f) * 8;
                if (p.words) copy8_async(to, blk < p.blocks ? src : p.scales, blk < p.blocks ? 8u : 0u);
                else {
                    uint2 v = make_uint2(0u, 0u);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (blk + j < p.blocks) { const uint32_t E = (uint32_t)__ldg(src + j) << (8 * (j & 3)); if (j < 4) v.x |= E; else v.y |= E; }
                    *(uint2*)to = v;
                }
            }
            // A warp brings a token's share of a box, a lane eight columns; float16 values are copied as they are, of others four boxes are asked for
            // before the first is used.
            const int units = len * p.wk * p.M;
            int q0 = warp;
            if (!SCALED && p.a_vec) {
                for (; q0 < units; q0 += warps) {
                    const int box = q0 / p.M, share = box / len, f = box - share * len, token = q0 - box * p.M;
                    const int k = (s_begin + share * per + f0 + f) * SLOT_K + lane * 8;
                    uint4* to = xs + (share * p.phase + f) * BOX_X + (lane >> 2) * BLOCK_X + token * 4 + (lane & 3);
                    if (k < p.K && k + 8 > p.K) *to = load_raw(p, token, k).a;
                    else copy16_async(to, k < p.K ? (const h16*)p.a + token * p.lda + k : (const h16*)p.a, k < p.K ? 16u : 0u);
                }
            }
            for (; q0 < units; q0 += 4 * warps) {
                Raw raw[4];
                int at[4], tok[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int q = min(q0 + j * warps, units - 1), box = q / p.M, share = box / len;
                    tok[j] = q - box * p.M;
                    at[j] = share * p.phase + box - share * len;
                    raw[j] = load_raw(p, tok[j], (s_begin + share * per + f0 + box - share * len) * SLOT_K + lane * 8);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (q0 + j * warps >= units) break;
                    uint4 v[TERMS];
                    float scale;
                    make_terms<TERMS, SCALED>(p, raw[j], v, scale);
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) xs[k * term_step + at[j] * BOX_X + (lane >> 2) * BLOCK_X + tok[j] * 4 + (lane & 3)] = v[k];
                    if (SCALED && lane == 0) sx[at[j] * (NT * 8) + tok[j]] = scale;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory");
            const int last = min(e, b + f0 + len);
            uint32_t xb = smem_u32(xs) + (uint32_t)(wk * p.phase * BOX_X + lane) * 16u;
            uint32_t sxb = smem_u32(sx) + (uint32_t)(wk * p.phase * (NT * 8) + 2 * t) * 4u;
            uint32_t swa = smem_u32(sw) + (uint32_t)((wf * 8 + g) * p.sw_ld + wk * p.phase * 8 + 2 * t);
            const uint32_t sw_half = (uint32_t)(8 * p.wf * p.sw_ld), x_term = (uint32_t)term_step * 16u;
            const uint32_t ring = smem_u32(smem) + (uint32_t)(wk * AHEAD * box_bytes + (wf * 8 + g) * 128 + t * 4), half = (uint32_t)box_bytes / 2;
#pragma unroll 1
            for (int s = b + f0; s < last; ++s, xb += BOX_X * 16, sxb += NT * 8 * 4, swa += 8) {
                // lane t: the scales of blocks 2t, 2t + 1 of its first row, then of its second
                const uint32_t two = lds16(swa) | lds16(swa + sw_half) << 16;
                float fs[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) fs[j] = scale_at(two, j);
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[wk][place], pass, p.err, 81));
                if (!ok) break;
                const uint32_t row = ring + (uint32_t)(place * box_bytes);
                uint32_t wa[SLOT_BLOCKS], wb[SLOT_BLOCKS];
#pragma unroll
                for (int i = 0; i < SLOT_BLOCKS; ++i) {
                    const uint32_t at = row + (uint32_t)((i ^ g) << 4);
                    wa[i] = lds32(at);
                    wb[i] = lds32(at + half);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[wk][place]);       // the box has been read
                if (++place == AHEAD) { place = 0; pass ^= 1u; }
                float sum[NT][4];
#pragma unroll
                for (int i = 0; i < SLOT_BLOCKS; ++i) {
                    uint32_t A[4], B[4];
                    codes_to_f16(wa[i], A);
                    codes_to_f16(wb[i], B);
                    const float ga = __shfl_sync(0xffffffffu, fs[i & 1], (lane & ~3) | (i >> 1));
                    const float gb = __shfl_sync(0xffffffffu, fs[2 + (i & 1)], (lane & ~3) | (i >> 1));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float c[4];
#pragma unroll
                        for (int k = 0; k < TERMS; ++k) {
                            const uint4 x = lds128(xb + k * x_term + (uint32_t)(i * BLOCK_X + n * 32) * 16u);
                            if (k == 0) mma_first(c, A[0], B[0], A[1], B[1], x.x, x.y);
                            else mma(c, A[0], B[0], A[1], B[1], x.x, x.y);
                            mma(c, A[2], B[2], A[3], B[3], x.z, x.w);
                        }
                        if (SCALED && i == 0) {
                            sum[n][0] = c[0] * ga; sum[n][1] = c[1] * ga; sum[n][2] = c[2] * gb; sum[n][3] = c[3] * gb;
                        } else {
                            float (&to)[4] = SCALED ? sum[n] : acc[n];
                            to[0] = fmaf(c[0], ga, to[0]); to[1] = fmaf(c[1], ga, to[1]); to[2] = fmaf(c[2], gb, to[2]); to[3] = fmaf(c[3], gb, to[3]);
                        }
                    }
                }
                if (SCALED) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 f = lds_f2(sxb + (uint32_t)n * 32u);
                        acc[n][0] = fmaf(sum[n][0], f.x, acc[n][0]); acc[n][1] = fmaf(sum[n][1], f.y, acc[n][1]);
                        acc[n][2] = fmaf(sum[n][2], f.x, acc[n][2]); acc[n][3] = fmaf(sum[n][3], f.y, acc[n][3]);
                    }
                }
            }
        }
    }
    if (!ok) {
        // A wait ran out: give copies in flight time to land before the shared memory is used otherwise.
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    // The shares' sums: [share][token][rows + 4], the lanes of a warp in 32 banks.  Gated: a warp's 8 gate rows stand in the first half of the rows,
    // its 8 up rows in the second; otherwise the two halves are neighbours.
    const int rows = p.wf * 16, ld = rows + 4;
    float* red = (float*)smem;
    __syncthreads();
    if (warp < warps) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int token = n * 8 + 2 * t + (j & 1);
                if (token < p.M) red[(wk * p.M + token) * ld + (j >> 1) * (rows / 2) + wf * 8 + g] = acc[n][j];
            }
    }
    const int splits = p.splits, rank = splits > 1 ? (int)cta_rank() : 0;
    if (splits > 1) cluster_sync(); else __syncthreads();
    auto total = [&](int token, int row) {                // shares in their order, then the cluster's blocks in theirs
        float v = 0.f;
        const float* at = red + token * ld + row;
        if (splits == 1) {
            for (int w = 0; w < p.wk; ++w) v += at[w * p.M * ld];
        } else
            for (int s = 0; s < splits; ++s)
                for (int w = 0; w < p.wk; ++w) v += ld_cluster(at + w * p.M * ld, (uint32_t)s);
        return v;
    };
    auto sum_of = [&](int token, int row, int w_row) {
        const float v = total(token, row);
        if (!SCALED || fabsf(v) < INFINITY) return v;
        const long long wb = (long long)w_row * p.blocks, ab = (long long)token * p.blocks;
        const char* a = (const char*)p.a + (p.a_kind == 2 ? ab * 16 : token * p.lda * (p.a_kind ? 4 : 2));
        return sum_again(v, p.codes + wb * 16, p.scales + wb, a, p.a_scales + ab, p.a_kind, p.K);
    };
    const int feats = p.gated ? rows / 2 : rows;
    const int f = threadIdx.x % feats;                    // a thread keeps its feature: blocks have at least as many threads as features
    const int n = first + f, groups = blockDim.x / feats;
    if ((int)threadIdx.x < groups * feats && n < p.N) {
        const float bias = p.bias ? __ldg(p.bias + n) : 0.f, bias_up = p.gated && p.bias ? __ldg(p.bias + p.N + n) : 0.f;
        for (int token = (threadIdx.x / feats) * splits + rank; token < p.M; token += groups * splits) {
            const long long o = (long long)token * p.ldc + n;
            const float res = p.residual ? __ldcg(p.residual + o) : 0.f;
            float v = mx_activation(sum_of(token, f, n) + bias, p.act);
            if (p.gated) v *= sum_of(token, feats + f, p.N + n) + bias_up;
            v += res;
            if (p.out_h16) ((h16*)p.out)[o] = float_to_h16(v);
            else ((float*)p.out)[o] = v;
        }
    }
    if (splits > 1) { __syncwarp(); cluster_sync(); }     // no block leaves while its sums may still be read
}

// ---- host -----------------------------------------------------------------------------------------
constexpr int SMEM_MOST = 224 * 1024;

bool map_codes(CUtensorMap* out, const void* ptr, int rows, int bytes, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)bytes};
    cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TERMS, int NT, bool SCALED>
int launch(const void* codes, const Params& p, int smem, cudaStream_t stream) {
    CUtensorMap map;
    if (!map_codes(&map, codes, p.w_rows, p.blocks * 16, 8 * p.wf)) return TNX_ERR_UNSUPPORTED;
    static TnxSmemLimit limit;
    auto kernel = gemv_kernel<TERMS, NT, SCALED>;
    const int r = limit.allow(kernel, SMEM_MOST);
    if (r) return r;
    const int per = (p.gated ? 8 : 16) * p.wf;
    const dim3 grid((p.N + per - 1) / per, 1, p.splits), block(32 * (p.wf * p.wk + 1));
    if (p.splits > 1) return tnx_launch_cluster(1, dim3(1, 1, p.splits), kernel, grid, block, smem, stream, map, p);
    return tnx_launch_ex(1, kernel, grid, block, smem, stream, map, p);
}
template <int TERMS, bool SCALED>
int launch_terms(const void* codes, const Params& p, int smem, cudaStream_t stream) {
    if (p.M <= 8) return launch<TERMS, 1, SCALED>(codes, p, smem, stream);
    return launch<TERMS, 2, SCALED>(codes, p, smem, stream);
}

int g_forced_wf = 0, g_forced_splits = 0;

}  // namespace

constexpr int FEW_TOKENS = 16;               // of a launch; more go in slices
// For tests: groups of 16 rows a block (1 to 15) and the split of K (1, 2, 4 or 8, where K allows it) whatever the sizes (0: the plan's own).
TNX_EXPORT int tnx_gemv_mxfp4_force(int wf, int splits) {
    if (wf < 0 || wf > MAX_WARPS || splits < 0 || splits > 8 || (splits & (splits - 1))) return TNX_ERR_BAD_ARG;
    g_forced_wf = wf; g_forced_splits = splits;
    return 0;
}

// a_kind: 0 16-bit, 1 32-bit activations (pitch lda), 2 codes (4-byte aligned) with a_scales; codes of W 16-byte aligned.
TNX_EXPORT int tnx_gemv_mxfp4(const void* a, int a_kind, const void* a_scales, long long lda, const void* codes, const void* scales, const float* bias,
                              const float* residual, void* out, int out_h16, long long ldc, int M, int N, int K, int act, int gated, int n_sms, int* err,
                              cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || a_kind < 0 || a_kind > 2 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0) return TNX_ERR_BAD_ARG;
    if (((uintptr_t)codes & 15) || (a_kind == 2 && ((uintptr_t)a & 3))) return TNX_ERR_UNSUPPORTED;
    if (M > FEW_TOKENS) {
        const long long blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
        for (int m = 0; m < M; m += FEW_TOKENS) {
            const void* a_m = a_kind == 2 ? (const void*)((const uint8_t*)a + m * blocks * 16) : (const void*)((const char*)a + m * lda * (a_kind ? 4 : 2));
            const int r = tnx_gemv_mxfp4(a_m, a_kind, a_scales ? (const void*)((const uint8_t*)a_scales + m * blocks) : nullptr, lda, codes, scales, bias,
                                         residual ? residual + m * ldc : nullptr, (void*)((char*)out + m * ldc * (out_h16 ? 2 : 4)), out_h16, ldc,
                                         M - m < FEW_TOKENS ? M - m : FEW_TOKENS, N, K, act, gated, n_sms, err, stream);
            if (r) return r;
        }
        return 0;
    }
    Params p;
    p.a = a; p.a_scales = (const uint8_t*)a_scales; p.lda = lda; p.a_kind = a_kind;
    p.a_vec = ((uintptr_t)a & 15) == 0 && lda % (a_kind == 1 ? 4 : 8) == 0;
    p.codes = (const uint8_t*)codes; p.scales = (const uint8_t*)scales; p.bias = bias; p.residual = residual; p.out = out; p.ldc = ldc; p.err = err;
    p.M = M; p.N = N; p.K = K; p.w_rows = gated ? 2 * N : N; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    p.slots = (p.blocks + SLOT_BLOCKS - 1) / SLOT_BLOCKS;
    p.act = act; p.out_h16 = out_h16; p.gated = gated;
    p.words = p.blocks % 8 == 0 && ((uintptr_t)scales & 7) == 0;
    const int terms = a_kind == 1 ? 3 : 1, groups = (N + (gated ? 8 : 16) - 1) / (gated ? 8 : 16);
    const int nt = M <= 8 ? 1 : 2;
    const int box_x = SLOT_K * 2 * nt * 8 * terms, box_s = nt * 8 * 4;      // shared memory of a box's activations, for one share of K
    auto scale_bytes = [&](int wf, int boxes) { return 16 * wf * ((boxes * 8 + 127) / 128 * 128 + 8); };        // eight rows lie in all banks
    auto phase_of = [&](int wf, int wk, int boxes) {                          // boxes a warp can take before its activations are replaced
        while (boxes > 1 && wf * wk * AHEAD * SLOT_BYTES + boxes * wk * (box_x + box_s) + scale_bytes(wf, boxes * wk) + 1024 > SMEM_MOST) --boxes;
        return boxes;
    };
    // The last plans by their sizes: working one out takes longer than a launch.
    struct Plan { int M, N, slots, gated, terms, sms, wf, wk, splits, sps; };
    static thread_local Plan known[64];
    Plan& k = known[((unsigned)M * 31u + (unsigned)N * 7u + (unsigned)p.slots * 13u + (unsigned)gated * 3u + (unsigned)terms) % 64u];
    const bool forced = g_forced_wf || g_forced_splits;
    if (!forced && k.M == M && k.N == N && k.slots == p.slots && k.gated == gated && k.terms == terms && k.sms == n_sms) {
        p.wf = k.wf; p.wk = k.wk; p.splits = k.splits; p.slots_per_split = k.sps;
    } else {
        // The busiest SM's boxes of codes, and what a block costs beside them (its activations, sums and barriers: as much as 16 boxes; activations that
        // come in two phases 12 more: 8 tokens by 2,048 x 4,096 12.8 us so, 8.3 by two parts of K in one phase each).
        long long best = -1;
        for (int splits = 1; splits <= 8; splits *= 2) {
            if (g_forced_splits && splits != g_forced_splits) continue;
            const int sps = (p.slots + splits - 1) / splits;
            if (splits > 1 && sps * (splits - 1) >= p.slots) continue;                 // no block without work
            for (int wf = 1; wf <= MAX_WARPS; ++wf) {
                if (g_forced_wf && wf != g_forced_wf) continue;
                int wk = MAX_WARPS / wf;
                if (wk > sps) wk = sps;
                auto least = [&]() { return wk * (wf * AHEAD * SLOT_BYTES + box_x + box_s) + scale_bytes(wf, wk) + 1024; };
                while (wk > 1 && least() > SMEM_MOST) --wk;
                if (least() > SMEM_MOST) continue;
                const long long blocks = (long long)((groups + wf - 1) / wf) * splits;
                // clusters of four find places on nine SMs in ten at a time, of eight on seven
                const int places = splits <= 2 ? n_sms : splits == 4 ? n_sms * 9 / 10 : n_sms * 7 / 10;
                const long long rounds = (blocks + places - 1) / places;
                const int each = (sps + wk - 1) / wk, phases = (each + phase_of(wf, wk, each) - 1) / phase_of(wf, wk, each);
                const long long cost = rounds * ((long long)wf * wk * each + 16 + 12 * (phases - 1) + (splits > 1 ? 8 : 0));
                if (best < 0 || cost < best) { best = cost; p.splits = splits; p.wf = wf; p.wk = wk; p.slots_per_split = sps; }
            }
        }
        if (best < 0) return TNX_ERR_UNSUPPORTED;
        if (!forced) k = {M, N, p.slots, gated, terms, n_sms, p.wf, p.wk, p.splits, p.slots_per_split};
    }
    const int ring = p.wf * p.wk * AHEAD * SLOT_BYTES;
    const int per = (p.slots_per_split + p.wk - 1) / p.wk;
    p.phase = phase_of(p.wf, p.wk, per);
    p.phase = (per + (per + p.phase - 1) / p.phase - 1) / ((per + p.phase - 1) / p.phase);           // as many phases, equal ones
    p.x_at = ring;
    p.sx_at = ring + p.phase * p.wk * box_x;
    const int sums = p.wk * M * (p.wf * 16 + 4) * 4, sx_end = p.sx_at + p.phase * p.wk * box_s;
    p.sw_at = sx_end;
    p.sw_ld = scale_bytes(1, p.phase * p.wk) / 16;
    const int used = sx_end + scale_bytes(p.wf, p.phase * p.wk);
    const int smem = (used > sums ? used : sums) + 1024;
    if (terms == 3) return launch_terms<3, true>(codes, p, smem, stream);
#ifdef TNX_F16
    if (a_kind == 0) return launch_terms<1, false>(codes, p, smem, stream);
#endif
    return launch_terms<1, true>(codes, p, smem, stream);
}

// The same with the parameters in one array (the stream last): a call through ctypes costs 0.1 us a parameter.
TNX_EXPORT int tnx_gemv_mxfp4_packed(const long long* v) {
    return tnx_gemv_mxfp4((const void*)v[0], (int)v[1], (const void*)v[2], (long long)v[3], (const void*)v[4], (const void*)v[5], (const float*)v[6],
                          (const float*)v[7], (void*)v[8], (int)v[9], (long long)v[10], (int)v[11], (int)v[12], (int)v[13], (int)v[14], (int)v[15],
                          (int)v[16], (int*)v[17], (cudaStream_t)v[18]);
}
