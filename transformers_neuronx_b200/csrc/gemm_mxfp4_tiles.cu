// Products of many tokens with a 4-bit matrix on the 5th-generation tensor cores (what is computed: gemm_mxfp4.cu).
//
// Persistent CTAs, one an SM, walk over tiles of 128 rows of W (the lanes of an accumulator) by up to 192 tokens (its columns).  Two accumulators:
// while one is written out by four warps of their own, the MMAs fill the other.  (A CTA a tile, whose sums went through shared memory,
// spent 11 us a tile outside of its main loop: 2,048 tokens by 16,384 x 4,096 229 us with 16-bit activations, 153 with 4-bit ones.)
// Sums go straight from tensor memory to memory: a warp's lanes are 32 neighbouring features, so that a token's store is 64 or 128 bytes.
// Gated tiles hold 16 gate rows and their 16 up rows for each of the four warps: gate and up values meet by one exchange of lanes 16 apart.
//
// gemm16 (16-bit activations): codes come through TMA, 256 columns of K a box; sixteen warps turn them into 16-bit values in tensor memory, 64 columns a
// group of four warps; the MMAs take them from there as their A operand, activations from shared memory.
// gemm4 (4-bit activations): both operands' codes come through TMA and are multiplied as they are (kind::mxf4); eight warps bring the scales to tensor
// memory.
#include "gemm_mxfp4.cuh"

namespace {

constexpr int MAX_BN = 192;                  // two accumulators and the operands' (or scales') stages are a tensor memory's 512 columns

struct Params {
    Epilogue e;
    const uint8_t* scales;
    const uint8_t* a_scales;                 // gemm4
    int w_rows, blocks;
    int num;                                 // stages of K a tile
    int tiles_t, tiles, bn;                  // tiles of tokens, tiles in all, tokens of a tile (a multiple of 16)
    int* err;
};

// Row `r` of the 128 of tile tw in W; rows behind the last count as the last one (their sums are not written).
__device__ __forceinline__ int tile_row(const Params& p, int tw, int r) {
    int row;
    if (!p.e.gated) row = tw * TILE_W + r;
    else row = tw * 64 + (r >> 5) * 16 + (r & 15) + ((r & 16) ? p.e.N : 0);
    return row < p.w_rows ? row : p.w_rows - 1;
}
// A box of 256 columns of tile tw's codes from column x (bytes) on.
__device__ __forceinline__ void load_codes(const Params& p, uint8_t* at, const CUtensorMap* map, uint64_t* bar, int x, int tw) {
    if (!p.e.gated) {
        tma_load_2d(at, map, bar, x, tw * TILE_W);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            tma_load_2d(at + q * 4096, map, bar, x, tw * 64 + q * 16);
            tma_load_2d(at + q * 4096 + 2048, map, bar, x, p.e.N + tw * 64 + q * 16);
        }
    }
}

// Sixteen columns (tokens from `token` on) of this lane's row.
template <int ACT>
__device__ __forceinline__ float act_of(float v, int act) { return ACT == TNX_ACT_COUNT ? apply_activation(v, act) : activate(v, ACT); }

__device__ __forceinline__ void put(void* at, float v, int h16_out) {
    if (h16_out) *(h16*)at = float_to_h16(v);
    else *(float*)at = v;
}

// WHOLE: all of the columns are tokens and all of the warp's rows features: no comparisons, and an address is one addition.
template <int ACT, bool WHOLE, bool H16, bool RESIDUAL>
__device__ __forceinline__ void write16_as(const Epilogue& e, const float (&v)[16], int n, int token, float bias) {
    const long long step = e.ldc * (H16 ? 2 : 4), o = (long long)token * e.ldc + n;
    const int tokens = e.M - token;
    float res[16];
    if (RESIDUAL) {
        const char* at = (const char*)(e.residual + o);
#pragma unroll
        for (int j = 0; j < 16; ++j, at += step) res[j] = WHOLE || j < tokens ? __ldcg((const float*)at) : 0.f;
    }
    char* at = (char*)e.out + o * (H16 ? 2 : 4);
#pragma unroll
    for (int j = 0; j < 16; ++j, at += step) {
        float r = act_of<ACT>(v[j] + bias, e.act);
        if (RESIDUAL) r += res[j];
        if (WHOLE || j < tokens) put(at, r, H16);
    }
}

template <int ACT>
__device__ __forceinline__ void write16(const Epilogue& e, const float (&v)[16], int n, int token, float bias, float bias_up) {
    const int lane = threadIdx.x & 31;
    if (e.gated) {
        const bool low = lane < 16;
        const long long step = 2 * e.ldc * (e.out_h16 ? 2 : 4);
        const int tokens = n < e.N ? e.M - token - (low ? 0 : 1) : 0;
        char* at = (char*)e.out + ((long long)(token + (low ? 0 : 1)) * e.ldc + n) * (e.out_h16 ? 2 : 4);
#pragma unroll
        for (int j = 0; j < 16; j += 2, at += step) {
            const float other = __shfl_xor_sync(0xffffffffu, low ? v[j + 1] : v[j], 16);
            const float gate = (low ? v[j] : other) + bias, up = (low ? other : v[j + 1]) + bias_up;
            const float r = act_of<ACT>(gate, e.act) * up;
            if (j < tokens) put(at, r, e.out_h16);
        }
        return;
    }
    if (n >= e.N) return;
    const bool whole = token + 16 <= e.M;
    if (e.out_h16) {
        if (whole) write16_as<ACT, true, true, false>(e, v, n, token, bias);
        else write16_as<ACT, false, true, false>(e, v, n, token, bias);
    } else if (e.residual) {
        if (whole) write16_as<ACT, true, false, true>(e, v, n, token, bias);
        else write16_as<ACT, false, false, true>(e, v, n, token, bias);
    } else {
        if (whole) write16_as<ACT, true, false, false>(e, v, n, token, bias);
        else write16_as<ACT, false, false, false>(e, v, n, token, bias);
    }
}

struct Rings {                               // both kernels' barriers between MMAs and epilogue
    uint64_t full[2], empty[2];
};

// The epilogue's warps, SETS of four, take sixteen columns in turn: accumulator `it & 1` of the CTA's it-th tile.
template <int SETS, typename Factor>
__device__ __forceinline__ bool epilogue(const Params& p, Rings& d, uint32_t tmem_d, int step, int set, Factor factor_of) {
    const int quad = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, r = quad * 32 + lane;
    bool ok = true;
    int it = 0;
    for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++it) {
        const int tt = tile % p.tiles_t, tw = tile / p.tiles_t, buf = it & 1;
        const int n = p.e.gated ? tw * 64 + quad * 16 + (lane & 15) : tw * TILE_W + r;
        float bias = 0.f, bias_up = 0.f;
        if (p.e.bias && n < p.e.N) {
            bias = __ldg(p.e.bias + n);
            if (p.e.gated) bias_up = __ldg(p.e.bias + p.e.N + n);
        }
        const float factor = factor_of(it);
        ok = __all_sync(0xffffffffu, mbar_wait(&d.full[buf], (uint32_t)(it >> 1) & 1u, p.err, 91));
        if (!ok) break;
        tc_fence_after();
        const uint32_t at = tmem_d + (uint32_t)(buf * step) + ((uint32_t)(quad * 32) << 16);
        const int token0 = tt * p.bn, cols = min(p.bn, (p.e.M - token0 + 15) & ~15);
        uint32_t raw[32];
        const int c0 = set * 16;
        if (c0 < cols) tmem_ld16(at + (uint32_t)c0, raw);
#pragma unroll 1
        for (int c = c0; c < cols; c += 16 * SETS) {
            tmem_ld_wait();
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(raw[j]) * factor;
            if (c + 16 * SETS < cols) tmem_ld16(at + (uint32_t)(c + 16 * SETS), raw);               // on its way while these are written
            switch (p.e.act) {
                case TNX_ACT_NONE: write16<TNX_ACT_NONE>(p.e, v, n, token0 + c, bias, bias_up); break;
                case TNX_ACT_RELU: write16<TNX_ACT_RELU>(p.e, v, n, token0 + c, bias, bias_up); break;
                case TNX_ACT_SILU: write16<TNX_ACT_SILU>(p.e, v, n, token0 + c, bias, bias_up); break;
                case TNX_ACT_GELU_NEW: write16<TNX_ACT_GELU_NEW>(p.e, v, n, token0 + c, bias, bias_up); break;
                default: write16<TNX_ACT_COUNT>(p.e, v, n, token0 + c, bias, bias_up);
            }
            __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d.empty[buf]);
    }
    return ok;
}

__device__ __forceinline__ void teardown(bool ok, uint32_t tmem, int warp) {
    if (!ok) {
        // A wait ran out: give copies in flight time to land before the shared memory is released.
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 3) { tc_fence_after(); tmem_dealloc(tmem, 512u); }
}

// ---- 16-bit activations ------------------------------------------------------------------------------
constexpr int STAGES16 = 4, BOXES = 4, GROUPS = 4;
constexpr int THREADS16 = 256 + 128 * GROUPS;        // warps 0: activations, 1: MMAs, 2: codes, 3: rows' references, 4..7: epilogue, 8..23: values
constexpr int X16_BYTES = MAX_BN * KB * 2;
constexpr int SMEM16 = BOXES * CODE_BYTES + STAGES16 * X16_BYTES + 1024;

__global__ void __launch_bounds__(THREADS16, 1)
gemm16_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sW = smem;
    uint8_t* sX = smem + BOXES * CODE_BYTES;
    __shared__ uint64_t w_full[BOXES], w_empty[BOXES], full[STAGES16], empty[STAGES16];
    __shared__ Rings d;
    __shared__ uint32_t tmem_base_smem;
#ifdef TNX_F16
    __shared__ uint64_t ref_full[2], ref_empty[2];
    __shared__ int row_ref[2][TILE_W];
#endif
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int num = p.num, boxes = (num + 3) / 4;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < BOXES; ++i) { mbar_init(&w_full[i], 1); mbar_init(&w_empty[i], 4 * GROUPS); }
        for (int i = 0; i < STAGES16; ++i) { mbar_init(&full[i], 5); mbar_init(&empty[i], 1); }       // full: activations and four warps' values
        for (int i = 0; i < 2; ++i) { mbar_init(&d.full[i], 1); mbar_init(&d.empty[i], 4); }
#ifdef TNX_F16
        for (int i = 0; i < 2; ++i) { mbar_init(&ref_full[i], 1); mbar_init(&ref_empty[i], 4 + 4 * GROUPS); }
#endif
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_x) : "memory");
    }
    if (warp == 3) { tmem_alloc(&tmem_base_smem, 512u); tmem_relinquish(); }
    pdl_wait();                                           // codes, scales and activations may be the preceding kernel's
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // The whole of tensor memory is this CTA's, so it begins at column 0: addresses that the compiler knows.
    constexpr uint32_t tmem_d = 0u, tmem_a = 2 * MAX_BN;
    bool ok = tmem_base_smem == 0u;                       // never anything else
    if (!ok) {
        if (threadIdx.x == 0) atomicExch(p.err, 90);
    } else if (warp == 0) {
        if (lane == 0) {
            Ring<STAGES16> r;
            int n = 0;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x)
                for (int i = 0; i < num; ++i, ++n) {
                    if (n >= STAGES16) { ok = mbar_wait(&empty[r.slot], r.pass ^ 1u, p.err, 92); if (!ok) break; }
                    mbar_expect_tx(&full[r.slot], (uint32_t)(p.bn * KB * 2));
                    tma_load_2d(sX + r.slot * X16_BYTES, &map_x, &full[r.slot], i * KB, tile % p.tiles_t * p.bn);
                    r.next();
                }
        }
        __syncwarp();
    } else if (warp == 2) {
        if (lane == 0) {
            int n = 0;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x)
                for (int i = 0; i < boxes; ++i, ++n) {
                    const int s = n % BOXES;
                    if (n >= BOXES) { ok = mbar_wait(&w_empty[s], (uint32_t)(n / BOXES - 1) & 1u, p.err, 93); if (!ok) break; }
                    mbar_expect_tx(&w_full[s], CODE_BYTES);
                    load_codes(p, sW + s * CODE_BYTES, &map_w, &w_full[s], i * (CODE_K / 2), tile / p.tiles_t);
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        // Two stages a turn: a wait costs this warp 200 cycles even where the barrier is ready (it queues behind the MMAs issued before it), the
        // MMAs of a stage take 256 to 384; a wait and other turn's work for every stage took 600 to 700.
        const uint32_t idesc = idesc16(p.bn);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(sX));
        const int total = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * num;
        int i = 0, it = 0;
        for (int n0 = 0; n0 < total && ok; n0 += STAGES16) {
            const uint32_t pass = (uint32_t)(n0 / STAGES16) & 1u;
#pragma unroll
            for (int s0 = 0; s0 < STAGES16; s0 += 2) {
                if (n0 + s0 >= total || !ok) break;
                const bool both = n0 + s0 + 1 < total;
                ok = mbar_wait(&full[s0], pass, p.err, 95) && (!both || mbar_wait(&full[s0 + 1], pass, p.err, 96));
                ok = __all_sync(0xffffffffu, ok);
#pragma unroll
                for (int s = s0; s < s0 + 2; ++s) {
                    if (!ok || (s > s0 && !both)) break;
                    if (i == 0 && it >= 2) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&d.empty[it & 1], (uint32_t)((it >> 1) - 1) & 1u, p.err, 94));
                        if (!ok) break;
                    }
                    tc_fence_after();
                    if (elected()) {
                        const uint32_t acc = tmem_d + (it & 1 ? MAX_BN : 0);
#pragma unroll
                        for (int k = 0; k < KB / 16; ++k)
                            umma_a_tmem(acc, tmem_a + (uint32_t)(s * 32 + 8 * k), desc0 + (uint64_t)(s * (X16_BYTES >> 4) + 2 * k), idesc, (i > 0 || k > 0) ? 1u : 0u);
                        umma_commit(&empty[s]);
                        if (i == num - 1) umma_commit(&d.full[it & 1]);
                    }
                    __syncwarp();
                    if (++i == num) { i = 0; ++it; }
                }
            }
        }
    } else if (warp == 3) {
#ifdef TNX_F16
        // The largest scale of every row of the next tiles, which becomes a factor of the row's sums.
        int it = 0;
        const bool wide = p.blocks % 16 == 0 && ((uintptr_t)p.scales & 15) == 0;
        for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++it) {
            const int buf = it & 1, tw = tile / p.tiles_t;
            if (it >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&ref_empty[buf], (uint32_t)((it >> 1) - 1) & 1u, p.err, 97));
            if (!ok) break;
            for (int row = lane >> 2; row < TILE_W; row += 8) {
                const uint8_t* q = p.scales + (long long)tile_row(p, tw, row) * p.blocks;
                uint32_t m = 0u;
                auto take = [&](uint32_t w) {                         // four bytes; 255 (NaN) is no size
#pragma unroll
                    for (int k = 0; k < 4; ++k) { const uint32_t E = (w >> (8 * k)) & 255u; m = max(m, E == 255u ? 0u : E); }
                };
                if (wide)
                    for (int j = (lane & 3) * 16; j < p.blocks; j += 64) { const uint4 v = __ldg((const uint4*)(q + j)); take(v.x); take(v.y); take(v.z); take(v.w); }
                else
                    for (int j = lane & 3; j < p.blocks; j += 4) take((uint32_t)__ldg(q + j));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                if ((lane & 3) == 0) row_ref[buf][row] = (int)m;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ref_full[buf]);
        }
#endif
    } else if (warp < 8) {
        ok = epilogue<1>(p, d, tmem_d, MAX_BN, 0, [&](int it) {
#ifdef TNX_F16
            const int buf = it & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(&ref_full[buf], (uint32_t)(it >> 1) & 1u, p.err, 98))) return 0.f;
            const uint32_t E = (uint32_t)row_ref[buf][(warp & 3) * 32 + lane];
            __syncwarp();
            if (lane == 0) mbar_arrive(&ref_empty[buf]);
            return mx_scale(E) * (1.f / (float)(1 << MX_F16_TOP));
#else
            (void)it;
            return 1.f;
#endif
        });
    } else {
        // Values: a thread owns a row, group j takes K block j of every box.
        const int quad = warp & 3, group = (warp - 8) >> 2, r = quad * 32 + lane;
        const bool even = p.blocks % 2 == 0 && ((uintptr_t)p.scales & 1) == 0;
        // The two scales of this group's K block, asked for four boxes ahead (a trip to memory takes longer than a box), over the tiles' ends.
        int ptile = blockIdx.x, pbox = 0;
        const uint8_t* sc = p.scales + (long long)tile_row(p, ptile / p.tiles_t, r) * p.blocks;
        auto load_scales = [&]() -> uint32_t {
            if (ptile >= p.tiles) return 0u;
            const int b = pbox * 8 + 2 * group;
            uint32_t v = 0u;
            if (b < p.blocks) v = even ? __ldg((const uint16_t*)(sc + b)) : (uint32_t)__ldg(sc + b) | (b + 1 < p.blocks ? (uint32_t)__ldg(sc + b + 1) << 8 : 0u);
            if (++pbox == boxes) {
                pbox = 0;
                ptile += gridDim.x;
                if (ptile < p.tiles) sc = p.scales + (long long)tile_row(p, ptile / p.tiles_t, r) * p.blocks;
            }
            return v;
        };
        uint32_t ahead[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ahead[j] = load_scales();
        const int total = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * boxes;
        int box = 0, it = 0, ref = 0;
        for (int g0 = 0; g0 < total && ok; g0 += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int g = g0 + u, ws = g % BOXES;
                if (g >= total || !ok) break;
                const uint32_t two = ahead[u];
                ahead[u] = load_scales();
#ifdef TNX_F16
                if (box == 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&ref_full[it & 1], (uint32_t)(it >> 1) & 1u, p.err, 99));
                    if (!ok) break;
                    ref = row_ref[it & 1][r];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ref_empty[it & 1]);
                }
#endif
                ok = __all_sync(0xffffffffu, mbar_wait(&w_full[ws], (uint32_t)(g / BOXES) & 1u, p.err, 100));
                if (!ok) break;
                const int i = box * 4 + group, n = it * num + i;
                if (++box == boxes) { box = 0; ++it; }
                uint32_t v[32];
                if (i < num) {
                    const uint32_t row_addr = smem_u32(sW + ws * CODE_BYTES) + (uint32_t)r * 128u;
                    uint4 q[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t at = row_addr + ((uint32_t)((2 * group + c) ^ (r & 7)) << 4);
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[c].x), "=r"(q[c].y), "=r"(q[c].z), "=r"(q[c].w) : "r"(at) : "memory");
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const MxValues t((two >> (8 * c)) & 255u, ref);
                        t.decode8(q[c].x, &v[16 * c]);
                        t.decode8(q[c].y, &v[16 * c + 4]);
                        t.decode8(q[c].z, &v[16 * c + 8]);
                        t.decode8(q[c].w, &v[16 * c + 12]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&w_empty[ws]);                 // this warp has read its share of the box
                if (i >= num) continue;
                const int s = n % STAGES16;
                if (n >= STAGES16) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (uint32_t)(n / STAGES16 - 1) & 1u, p.err, 101));
                    if (!ok) break;
                    tc_fence_after();
                }
                tmem_st32(tmem_a + (uint32_t)(s * 32) + ((uint32_t)(quad * 32) << 16), v);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
            }
        }
    }
    teardown(ok, tmem_base_smem, warp);
}

// ---- 4-bit activations -------------------------------------------------------------------------------
constexpr int STAGES4 = 5;
constexpr int THREADS4 = 640;                // warps 0: TMA, 1: MMAs, 4..11: epilogue, 12..19: scales
constexpr int X4_BYTES = MAX_BN * CODE_K / 2, STAGE4_BYTES = CODE_BYTES + X4_BYTES;
constexpr int SMEM4 = STAGES4 * STAGE4_BYTES + 1024;
constexpr int SF_COLS = 24;                  // a stage's scales: 2 x 4 columns for W, 2 x 8 for up to 256 tokens
constexpr int SF_LD = SF_COLS + 4;           // a lane's scales in shared memory: 16-byte loads of eight lanes lie in all banks

__device__ __forceinline__ void group_sync(int group) {
    if (group) asm volatile("bar.sync 2, 128;" ::: "memory");
    else asm volatile("bar.sync 1, 128;" ::: "memory");
}

__global__ void __launch_bounds__(THREADS4, 1)
gemm4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
    static_assert(2 * MAX_BN + STAGES4 * SF_COLS <= 512, "tensor memory");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[STAGES4], empty[STAGES4];
    __shared__ Rings d;
    __shared__ uint32_t tmem_base_smem;
    __shared__ __align__(16) uint32_t sf_smem[2][2][32 * SF_LD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int num = p.num;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES4; ++i) { mbar_init(&full[i], 5); mbar_init(&empty[i], 1); }         // full: codes and four warps' scales
        for (int i = 0; i < 2; ++i) { mbar_init(&d.full[i], 1); mbar_init(&d.empty[i], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_x) : "memory");
    }
    if (warp == 3) { tmem_alloc(&tmem_base_smem, 512u); tmem_relinquish(); }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem_d = 0u, tmem_sf = 2 * MAX_BN;            // the whole of tensor memory is this CTA's
    bool ok = tmem_base_smem == 0u;                       // never anything else
    if (!ok) {
        if (threadIdx.x == 0) atomicExch(p.err, 90);
    } else if (warp == 0) {
        if (lane == 0) {
            Ring<STAGES4> r;
            int n = 0;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x)
                for (int i = 0; i < num; ++i, ++n) {
                    if (n >= STAGES4) { ok = mbar_wait(&empty[r.slot], r.pass ^ 1u, p.err, 111); if (!ok) break; }
                    uint8_t* at = smem + r.slot * STAGE4_BYTES;
                    mbar_expect_tx(&full[r.slot], (uint32_t)(CODE_BYTES + p.bn * (CODE_K / 2)));
                    load_codes(p, at, &map_w, &full[r.slot], i * (CODE_K / 2), tile / p.tiles_t);
                    tma_load_2d(at + CODE_BYTES, &map_x, &full[r.slot], i * (CODE_K / 2), tile % p.tiles_t * p.bn);
                    r.next();
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc0 = idesc4(p.bn, 0), idesc2 = idesc4(p.bn, 2);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(smem));
        const int total = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * num;
        int i = 0, it = 0;
        Ring<STAGES4> r;
        for (int n = 0; n < total && ok; n += 2) {        // two stages a turn, as above
            Ring<STAGES4> q = r;
            q.next();
            const bool both = n + 1 < total;
            ok = mbar_wait(&full[r.slot], r.pass, p.err, 113) && (!both || mbar_wait(&full[q.slot], q.pass, p.err, 114));
            ok = __all_sync(0xffffffffu, ok);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!ok || (h && !both)) break;
                if (i == 0 && it >= 2) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&d.empty[it & 1], (uint32_t)((it >> 1) - 1) & 1u, p.err, 112));
                    if (!ok) break;
                }
                tc_fence_after();
                const uint64_t adesc = desc0 + (uint64_t)(r.slot * (STAGE4_BYTES >> 4)), bdesc = adesc + (uint64_t)(CODE_BYTES >> 4);
                const uint32_t sf = tmem_sf + (uint32_t)(r.slot * SF_COLS), acc = tmem_d + (it & 1 ? MAX_BN : 0);
                if (elected()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)           // 64 columns of K = 32 bytes = 2 units of the address field
                        umma_mxf4(acc, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), k & 1 ? idesc2 : idesc0, sf + 4u * (k >> 1),
                                  sf + 8u + 8u * (k >> 1), (i > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&empty[r.slot]);
                    if (i == num - 1) umma_commit(&d.full[it & 1]);
                }
                __syncwarp();
                r.next();
                if (++i == num) { i = 0; ++it; }
            }
        }
    } else if (warp >= 12) {
        // Scales: two groups of four warps take stages in turn; a thread loads a row of W's and up to two of the activations', eight scales each,
        // three turns ahead (a trip to memory takes longer than a stage); they meet in shared memory, whence every warp takes all of them
        // to the lanes of its quarter.
        const int quad = warp & 3, group = (warp - 12) >> 2, r = quad * 32 + lane;
        const bool words = p.blocks % 8 == 0 && (((uintptr_t)p.scales | (uintptr_t)p.a_scales) & 7) == 0;        // eight scales are one aligned load
        const bool second = r + 128 < p.bn, first = r < p.bn;
        const uint8_t* w_end = p.scales + (long long)p.w_rows * p.blocks;
        const uint8_t* x_end = p.a_scales + (long long)p.e.M * p.blocks;
        struct Scales { uint2 w, x[2]; };
        int ptile = blockIdx.x, pi = group;
        const uint8_t *ws = nullptr, *xs0 = nullptr, *xs1 = nullptr;
        auto aim = [&]() {                                // over the tiles' ends
            while (pi >= num) { pi -= num; ptile += gridDim.x; }
            if (ptile >= p.tiles) return;
            const int token = ptile % p.tiles_t * p.bn + r;
            ws = p.scales + (long long)tile_row(p, ptile / p.tiles_t, r) * p.blocks + pi * 8;
            xs0 = p.a_scales + (long long)min(token, p.e.M - 1) * p.blocks + pi * 8;
            xs1 = p.a_scales + (long long)min(token + 128, p.e.M - 1) * p.blocks + pi * 8;
        };
        auto load = [&]() {
            Scales q;
            q.w = q.x[0] = q.x[1] = make_uint2(0u, 0u);
            if (ptile >= p.tiles) return q;
            if (words) {
                q.w = __ldg((const uint2*)ws);
                if (first) q.x[0] = __ldg((const uint2*)xs0);
                if (second) q.x[1] = __ldg((const uint2*)xs1);
            } else {
                const int n = p.blocks - pi * 8;
                q.w = load8(ws, p.scales, w_end, n);
                if (first) q.x[0] = load8(xs0, p.a_scales, x_end, n);
                if (second) q.x[1] = load8(xs1, p.a_scales, x_end, n);
            }
            pi += 2; ws += 16; xs0 += 16; xs1 += 16;
            if (pi >= num) aim();
            return q;
        };
        aim();
        Scales ahead[3] = {load(), load(), load()};
        const int total = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * num;
        int turn = 0, s = group;
        uint32_t pass = 1u;                               // of the stage's last use, from its second use on
        for (int i0 = group; i0 < total; i0 += 6) {       // whole even if a wait ran out: the groups' warps meet at their barrier
#pragma unroll
            for (int u = 0; u < 3; ++u) {                 // (unrolled so that a register waits for its load where it is used)
                const int i = i0 + 2 * u;
                if (i >= total) break;
                const Scales now = ahead[u];
                ahead[u] = load();
                uint32_t* buf = &sf_smem[group][turn][0]; // two in turn: one barrier a stage
                turn ^= 1;
                uint32_t* mine = buf + lane * SF_LD + quad;
                mine[0] = now.w.x; mine[4] = now.w.y;
                mine[8] = now.x[0].x; mine[16] = now.x[0].y;
                mine[12] = now.x[1].x; mine[20] = now.x[1].y;
                group_sync(group);
                uint32_t v[SF_COLS];
#pragma unroll
                for (int c = 0; c < SF_COLS; c += 4) {
                    const uint4 q = *(const uint4*)(buf + lane * SF_LD + c);
                    v[c] = q.x; v[c + 1] = q.y; v[c + 2] = q.z; v[c + 3] = q.w;
                }
                if (ok && i >= STAGES4) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], pass, p.err, 115));
                    tc_fence_after();
                }
                if (ok) {
                    const uint32_t at = tmem_sf + (uint32_t)(s * SF_COLS) + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                    for (int c = 0; c < SF_COLS; c += 8) {
                        uint32_t q[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) q[j] = v[c + j];
                        tmem_st8(at + (uint32_t)c, q);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[s]);
                }
                s += 2;
                if (s >= STAGES4) { s -= STAGES4; pass ^= 1u; }
            }
        }
    } else if (warp >= 4) {
        ok = epilogue<2>(p, d, tmem_d, MAX_BN, (warp - 4) >> 2, [](int) { return 1.f; });
    }
    teardown(ok, tmem_base_smem, warp);
}

// ---- host -----------------------------------------------------------------------------------------
int g_forced_bn = 0;

// Tokens of a tile: the busiest CTA's rounds of tiles, each as long as its columns and what a stage costs whatever its columns are, `extra` of them.
void plan(Params& p, int n_sms, int tiles_w, int extra) {
    long long best = -1;
    const int most = (p.e.M + 15) / 16 * 16;
    for (int bn = MAX_BN; bn >= 64; bn -= 16) {
        if (g_forced_bn && bn != g_forced_bn) continue;
        if (bn > most && bn > 64 && !g_forced_bn) continue;
        const int tt = (p.e.M + bn - 1) / bn;
        const long long rounds = ((long long)tt * tiles_w + n_sms - 1) / n_sms, cost = rounds * (bn + extra);
        if (best < 0 || cost < best) { best = cost; p.bn = bn; p.tiles_t = tt; p.tiles = tt * tiles_w; }
    }
}

template <typename Kernel>
int launch(Kernel kernel, TnxSmemLimit& limit, int threads, int smem, const CUtensorMap& mw, const CUtensorMap& mx, const Params& p, int n_sms, cudaStream_t stream) {
    const int r = limit.allow(kernel, smem);
    if (r) return r;
    return tnx_launch_ex(1, kernel, dim3(p.tiles < n_sms ? p.tiles : n_sms), dim3(threads), smem, stream, mw, mx, p);
}

}  // namespace

// For sweeps: the tokens of a tile (a multiple of 16 from 64 to 192) whatever the sizes (0: the plan's own).
TNX_EXPORT void tnx_gemm_mxfp4_tiles_force(int bn) { g_forced_bn = bn; }

// 16-bit activations [M, K] (pitch lda, a multiple of 8 elements, 16-byte aligned) by codes [w_rows][blocks * 16] (16-byte aligned).
TNX_EXPORT int tnx_gemm_mxfp4_tiles_16(const void* a, long long lda, const void* codes, const void* scales, const float* bias, const float* residual, void* out,
                                       int out_h16, long long ldc, int M, int N, int K, int act, int gated, int n_sms, int* err, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0) return TNX_ERR_BAD_ARG;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    if (lda % 8 || ((uintptr_t)a & 15) || ((uintptr_t)codes & 15) || (long long)tiles_w * ((M + 63) / 64) > 0x3FFFFFFF) return TNX_ERR_UNSUPPORTED;
    Params p;
    fill_epilogue(p.e, bias, residual, out, out_h16, ldc, M, N, act, gated);
    p.scales = (const uint8_t*)scales; p.a_scales = nullptr; p.err = err;
    p.w_rows = gated ? 2 * N : N; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK; p.num = (K + KB - 1) / KB;
    plan(p, n_sms, tiles_w, 400);
    CUtensorMap mw, mx;
    if (!map_bytes(&mw, codes, p.w_rows, p.blocks * 16, gated ? 16 : TILE_W) || !map_h16(&mx, a, M, K, lda, p.bn)) return TNX_ERR_UNSUPPORTED;
    static TnxSmemLimit limit;
    return launch(gemm16_kernel, limit, THREADS16, SMEM16, mw, mx, p, n_sms, stream);
}

// 4-bit activations: codes [M][blocks * 16] (16-byte aligned) and scales [M][blocks].
TNX_EXPORT int tnx_gemm_mxfp4_tiles_4(const void* a, const void* a_scales, const void* codes, const void* scales, const float* bias, const float* residual,
                                      void* out, int out_h16, long long ldc, int M, int N, int K, int act, int gated, int n_sms, int* err, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0) return TNX_ERR_BAD_ARG;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    if (((uintptr_t)a & 15) || ((uintptr_t)codes & 15) || (long long)tiles_w * ((M + 63) / 64) > 0x3FFFFFFF) return TNX_ERR_UNSUPPORTED;
    Params p;
    fill_epilogue(p.e, bias, residual, out, out_h16, ldc, M, N, act, gated);
    p.scales = (const uint8_t*)scales; p.a_scales = (const uint8_t*)a_scales; p.err = err;
    p.w_rows = gated ? 2 * N : N; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK; p.num = (K + CODE_K - 1) / CODE_K;
    plan(p, n_sms, tiles_w, 400);
    CUtensorMap mw, mx;
    if (!map_bytes(&mw, codes, p.w_rows, p.blocks * 16, gated ? 16 : TILE_W) || !map_bytes(&mx, a, M, p.blocks * 16, p.bn)) return TNX_ERR_UNSUPPORTED;
    static TnxSmemLimit limit;
    return launch(gemm4_kernel, limit, THREADS4, SMEM4, mw, mx, p, n_sms, stream);
}
