// Products of many tokens with a 4-bit matrix on the 5th-generation tensor cores (what is computed: gemm_mxfp4.cu).
//
// Persistent CTAs, one an SM, walk over tiles of 128 rows of W (the lanes of an accumulator) by up to 192 tokens (its columns).  Two accumulators:
// while one is written out by warps of their own, the MMAs fill the other.  (A CTA a tile, whose sums went through shared memory, spent 11 us a tile
// outside of its main loop.)  2,048 tokens by 16,384 x 4,096: 223 to 240 us with 16-bit activations, 1.15 to 1.23 PFLOP/s, where the tensor cores are busy
// for 61% of the time at 1.6 GHz, which the power limit leaves (275 when run for seconds, 1 PFLOP/s; of 227, 186 or 171 are left without MMAs, 195 or 211
// without decoding, 121 without either: what the activations' way from L2 takes); 69 to 73 us with 4-bit ones, 3.8 to 4 PFLOP/s, of which the loads alone
// take 56.
// Sums go straight from tensor memory to memory: a warp's lanes are 32 neighbouring features, so that a token's store is 64 or 128 bytes.
// Gated tiles alternate eight gate rows and their eight up rows: gate and up values meet by one exchange of lanes eight apart.
//
// gemm16 (16-bit activations): codes come through TMA, 256 columns of K a box; sixteen warps turn them into 16-bit values in tensor memory, 64 columns a
// group of four warps; the MMAs take them from there as their A operand, activations from shared memory.
// gemm4 (4-bit activations): both operands' codes come through TMA and are multiplied as they are (kind::mxf4); so do the scales, which a kernel before
// this one has put into the order in which they are copied on to tensor memory.
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
    int one_box;                             // gated: a tile's gate and up rows are one box of a map of four dimensions
    int* err;
};

// Row `r` of the 128 of tile tw in W; rows behind the last count as the last one (their sums are not written).
__device__ __forceinline__ int tile_row(const Params& p, int tw, int r) {
    int row;
    if (!p.e.gated) row = tw * TILE_W + r;
    else row = tw * 64 + (r >> 4) * 8 + (r & 7) + ((r & 8) ? p.e.N : 0);
    return row < p.w_rows ? row : p.w_rows - 1;
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(smem_u32(dst)), "l"((unsigned long long)map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// A box of 256 columns of tile tw's codes from column x (bytes) on.
__device__ __forceinline__ void load_codes(const Params& p, uint8_t* at, const CUtensorMap* map, uint64_t* bar, int x, int tw) {
    if (!p.e.gated) tma_load_2d(at, map, bar, x, tw * TILE_W);
    else if (p.one_box) tma_load_4d(at, map, bar, x, 0, 0, tw * 8);
    else
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
            tma_load_2d(at + q * 2048, map, bar, x, tw * 64 + q * 8);
            tma_load_2d(at + q * 2048 + 1024, map, bar, x, p.e.N + tw * 64 + q * 8);
        }
}

// ACT: an activation known to the compiler, or TNX_ACT_COUNT: any, by its number and in full precision.
template <int ACT>
__device__ __forceinline__ float act_of(float v, int act) { return ACT == TNX_ACT_COUNT ? mx_activation(v, act) : activate(v, ACT); }

__device__ __forceinline__ void put(void* at, float v, int h16_out) {
    if (h16_out) *(h16*)at = float_to_h16(v);
    else *(float*)at = v;
}

// Sixteen columns (tokens from `token` on) of this lane's row.  WHOLE: all of the columns are tokens and all of the warp's rows features: no
// comparisons, and an address is one addition.
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
        const bool low = !(lane & 8);
        const long long step = 2 * e.ldc * (e.out_h16 ? 2 : 4);
        const int tokens = n < e.N ? e.M - token - (low ? 0 : 1) : 0;
        char* at = (char*)e.out + ((long long)(token + (low ? 0 : 1)) * e.ldc + n) * (e.out_h16 ? 2 : 4);
#pragma unroll
        for (int j = 0; j < 16; j += 2, at += step) {
            const float other = __shfl_xor_sync(0xffffffffu, low ? v[j + 1] : v[j], 8);
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

// Two warps issue the MMAs, a stage each in turn: a warp's waits for a stage cost 200 to 250 cycles even where the barriers are ready (they queue behind
// the MMAs that it issued before), which the other one's MMAs then cover.  The turn is handed on when a stage's MMAs have been issued, so they are
// carried out in the order of the stages.  (Also by a warp whose wait ran out: the other one must not wait for ever.)
__device__ __forceinline__ void await_turn(int who) { asm volatile("bar.sync %0, 64;" ::"r"(2 + who) : "memory"); tc_fence_after(); }
__device__ __forceinline__ void hand_on(int who) { tc_fence_before(); __syncwarp(); asm volatile("bar.arrive %0, 64;" ::"r"(3 - who) : "memory"); }

struct Rings {                               // both kernels' barriers between MMAs and epilogue; full: one arrival from either warp of the MMAs
    uint64_t full[2], empty[2];
};

// The epilogue's warps, SETS of four, take sixteen columns in turn: accumulator `it & 1` of the CTA's it-th tile.
template <int SETS, typename Factor>
__device__ __forceinline__ bool epilogue(const Params& p, Rings& d, uint32_t tmem_d, int step, int set, Factor factor_of) {
    const int quad = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, r = quad * 32 + lane;
    // the few instructions' forms are for results that are rounded to 16 bits
    const int act = p.e.out_h16 || p.e.act == TNX_ACT_NONE || p.e.act == TNX_ACT_RELU ? p.e.act : TNX_ACT_COUNT;
    bool ok = true;
    int it = 0;
    for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++it) {
        const int tt = tile % p.tiles_t, tw = tile / p.tiles_t, buf = it & 1;
        const int n = p.e.gated ? tw * 64 + quad * 16 + (lane >> 4) * 8 + (lane & 7) : tw * TILE_W + r;
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
            switch (act) {
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
constexpr int BOXES = 4, GROUPS = 4;          // boxes of codes in flight; groups of four warps, one for each of a box's four K blocks
constexpr int PARTS = 2, X_STAGES = 3;       // K blocks a stage; stages of activations (of values, in tensor memory: a K block a group)
constexpr int THREADS16 = 256 + 128 * GROUPS;        // warps 0: activations, 1, 3: MMAs, 2: codes, 4..7: rows' references and epilogue, 8..23: values
constexpr int X16_BYTES = MAX_BN * KB * 2;   // of a K block
constexpr int SMEM16 = BOXES * CODE_BYTES + X_STAGES * PARTS * X16_BYTES + 1024;

__global__ void __launch_bounds__(THREADS16, 1)
gemm16_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sW = smem;
    uint8_t* sX = smem + BOXES * CODE_BYTES;
    __shared__ uint64_t w_full[BOXES], w_empty[BOXES], x_full[X_STAGES], x_empty[X_STAGES], a_full[GROUPS / PARTS], a_empty[GROUPS];
    __shared__ Rings d;
    __shared__ uint32_t tmem_base_smem;
#ifdef TNX_F16
    __shared__ uint64_t ref_full[2], ref_empty[2];
    __shared__ int row_ref[2][TILE_W];
#endif
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int num = p.num, stages = (num + PARTS - 1) / PARTS, boxes = (num + 3) / 4;             // K blocks, stages and boxes a tile

    if (threadIdx.x == 0) {
        for (int i = 0; i < BOXES; ++i) { mbar_init(&w_full[i], 1); mbar_init(&w_empty[i], 4 * GROUPS); }
        for (int i = 0; i < X_STAGES; ++i) { mbar_init(&x_full[i], 1); mbar_init(&x_empty[i], 1); }
        for (int i = 0; i < GROUPS; ++i) mbar_init(&a_empty[i], 1);
        for (int i = 0; i < GROUPS / PARTS; ++i) mbar_init(&a_full[i], 4 * PARTS);
        for (int i = 0; i < 2; ++i) { mbar_init(&d.full[i], 2); mbar_init(&d.empty[i], 4); }
#ifdef TNX_F16
        for (int i = 0; i < 2; ++i) { mbar_init(&ref_full[i], 4); mbar_init(&ref_empty[i], 4 * GROUPS); }
#endif
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_x) : "memory");
    }
    pdl_wait();                                           // codes, scales and activations may be the preceding kernel's
    if (warp == 3) { tmem_alloc(&tmem_base_smem, 512u); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();             // a kernel that started before all CTAs have their tensor memory might hold some and wait for them
    // The whole of tensor memory is this CTA's, so it begins at column 0: addresses that the compiler knows.
    constexpr uint32_t tmem_d = 0u, tmem_a = 2 * MAX_BN;
    bool ok = tmem_base_smem == 0u;                       // never anything else
    if (!ok) {
        if (threadIdx.x == 0) atomicExch(p.err, 90);
    } else if (warp == 0) {
        if (lane == 0) {
            Ring<X_STAGES> r;
            int n = 0;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
                const int token0 = tile % p.tiles_t * p.bn;
                for (int i = 0; i < stages; ++i, ++n) {
                    if (n >= X_STAGES) { ok = mbar_wait(&x_empty[r.slot], r.pass ^ 1u, p.err, 92); if (!ok) break; }
                    const int parts = min(PARTS, num - i * PARTS);
                    mbar_expect_tx(&x_full[r.slot], (uint32_t)(parts * p.bn * KB * 2));
                    for (int j = 0; j < parts; ++j)
                        tma_load_2d(sX + (r.slot * PARTS + j) * X16_BYTES, &map_x, &x_full[r.slot], (i * PARTS + j) * KB, token0);
                    r.next();
                }
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
    } else if (warp == 1 || warp == 3) {
        // A stage is 128 columns of K, eight MMAs.
        const int who = warp == 1 ? 0 : 1;
        const uint32_t idesc = idesc16(p.bn);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(sX));
        const int total = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * stages;
        Ring<X_STAGES> r;
        uint32_t passes = 0u;                             // of the places of values, a bit each
        int it = 0, i = 0;
        for (int n = 0; n < total; ++n) {
            const int place = i * PARTS % GROUPS, parts = min(PARTS, num - i * PARTS);
            if ((n & 1) == who) {
                // (a tile's last stage may have had the same place, so it has to be the turn of this one before its barrier tells anything)
                const bool early = i == 0 && n > 0;
                if (early) await_turn(who);
                if (ok && it >= 2 && i < 2) ok = mbar_wait(&d.empty[it & 1], (uint32_t)((it >> 1) - 1) & 1u, p.err, 94);
                ok = ok && mbar_wait(&x_full[r.slot], r.pass, p.err, 95) && mbar_wait(&a_full[place / PARTS], (passes >> place) & 1u, p.err, 96);
                ok = __all_sync(0xffffffffu, ok);
                if (n && !early) await_turn(who);
                tc_fence_after();
                const uint32_t acc = tmem_d + (it & 1 ? MAX_BN : 0);
                const uint64_t bdesc = desc0 + (uint64_t)(r.slot * (PARTS * X16_BYTES >> 4));
                const uint32_t a = tmem_a + (uint32_t)(place * 32);
                if (ok && elected()) {
#pragma unroll
                    for (int j = 0; j < PARTS; ++j) {
                        if (j < parts) {
#pragma unroll
                            for (int k = 0; k < KB / 16; ++k)
                                umma_a_tmem(acc, a + (uint32_t)(32 * j + 8 * k), bdesc + (uint64_t)(j * (X16_BYTES >> 4) + 2 * k), idesc, (i > 0 || j > 0 || k > 0) ? 1u : 0u);
                        }
                        umma_commit(&a_empty[place + j]);
                    }
                    umma_commit(&x_empty[r.slot]);
                    if (i >= stages - 2) umma_commit(&d.full[it & 1]);
                    if (stages == 1) umma_commit(&d.full[it & 1]);
                }
                __syncwarp();
                if (n + 1 < total) hand_on(who);
            }
            r.next();
            passes ^= 1u << place;
            if (++i == stages) { i = 0; ++it; }
        }
    } else if (warp < 8) {
#ifdef TNX_F16
        // The largest scale of every row of a tile, which becomes a factor of the row's sums: found two tiles ahead, each warp for the rows that it writes
        // out.
        const bool wide = p.blocks % 16 == 0 && ((uintptr_t)p.scales & 15) == 0;
        auto find_refs = [&](int it) {
            const int tile = (int)blockIdx.x + it * (int)gridDim.x, buf = it & 1, r0 = (warp & 3) * 32 + (lane >> 2);
            if (tile >= p.tiles) return;
            auto largest = [](uint32_t m, uint32_t w) {               // of four bytes; 255 (NaN) is no size
#pragma unroll
                for (int k = 0; k < 4; ++k) { const uint32_t E = (w >> (8 * k)) & 255u; m = max(m, E == 255u ? 0u : E); }
                return m;
            };
            // four rows of eight lanes' in flight at a time: the first tile waits for this
            const uint8_t* q[4];
            uint32_t m[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q[e] = p.scales + (long long)tile_row(p, tile / p.tiles_t, r0 + e * 8) * p.blocks;
                m[e] = 0u;
            }
            if (wide) {
#pragma unroll 2
                for (int j = (lane & 3) * 16; j < p.blocks; j += 64) {
                    uint4 v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __ldg((const uint4*)(q[e] + j));
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[e] = largest(largest(largest(largest(m[e], v[e].x), v[e].y), v[e].z), v[e].w);
                }
            } else {
#pragma unroll 2
                for (int j = lane & 3; j < p.blocks; j += 4) {
                    uint32_t v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __ldg(q[e] + j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[e] = max(m[e], v[e] == 255u ? 0u : v[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = max(m[e], __shfl_xor_sync(0xffffffffu, m[e], 1));
                m[e] = max(m[e], __shfl_xor_sync(0xffffffffu, m[e], 2));
                if ((lane & 3) == 0) row_ref[buf][r0 + e * 8] = (int)m[e];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ref_full[buf]);
        };
        find_refs(0);
        find_refs(1);
#endif
        ok = epilogue<1>(p, d, tmem_d, MAX_BN, 0, [&](int it) {
#ifdef TNX_F16
            const int buf = it & 1;
            const uint32_t E = (uint32_t)row_ref[buf][(warp & 3) * 32 + lane];
            __syncwarp();
            if (__all_sync(0xffffffffu, mbar_wait(&ref_empty[buf], (uint32_t)(it >> 1) & 1u, p.err, 97))) find_refs(it + 2);
            return mx_scale(E) * (1.f / (float)(1 << MX_F16_TOP));
#else
            (void)it;
            return 1.f;
#endif
        });
    } else {
        // Values: a thread owns a row, group j takes K block j of every box and keeps a place of its own in tensor memory, which is free as soon as that K
        // block's four MMAs are done.  (Places that the groups took in turn: a group that did not see all of a place's turns, of which a barrier tells
        // only every other apart, could overwrite values in use.)
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
        int box = 0, it = 0, ref = 0, use = 0;            // use: K blocks that this group has filled
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
                const bool has = box * 4 + group < num, stage = box * 4 + group / PARTS * PARTS < num;       // the tile's last box may end before them
                if (++box == boxes) { box = 0; ++it; }
                uint32_t v[32];
                if (has) {
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
                if (!stage) continue;
                if (use > 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&a_empty[group], (uint32_t)(use - 1) & 1u, p.err, 101));
                    if (!ok) break;
                    tc_fence_after();
                }
                ++use;
                if (has) {
                    tmem_st32(tmem_a + (uint32_t)(group * 32) + ((uint32_t)(quad * 32) << 16), v);
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[group / PARTS]);
            }
        }
    }
    teardown(ok, tmem_base_smem, warp);
}

// ---- 4-bit activations -------------------------------------------------------------------------------
constexpr int STAGES4 = 5;
constexpr int THREADS4 = 384;                // warps 0, 2: TMA, 1, 3: MMAs, 4..11: epilogue
constexpr int X4_BYTES = MAX_BN * CODE_K / 2, STAGE4_BYTES = CODE_BYTES + X4_BYTES;
constexpr int SF_ATOM = 512;                 // scales of 128 rows and 128 columns of K: [32 lanes][rows l, 32 + l, 64 + l, 96 + l][4 blocks]
constexpr int SFW_BYTES = 2 * SF_ATOM, SFX_BYTES = 4 * SF_ATOM;        // a stage's for W and for up to 256 tokens
constexpr int SMEM4 = STAGES4 * (STAGE4_BYTES + SFW_BYTES + SFX_BYTES) + 1024;
constexpr int SF_COLS = 24;                  // tensor memory of a stage's scales: 2 x 4 columns for W, 2 x 8 for up to 256 tokens

// The scales as the MMAs read them, from rows of bytes to atoms: W's for every tile and stage (1 KB), then the activations' (1 or 2 KB).  Gathered
// row by row by the product's own warps, eight bytes of 320 rows a stage, they were what the product waited for (2,048 tokens by
// 16,384 x 4,096: 103 us, 70 without them); here they are moved once, a warp's lanes side by side.
__global__ void __launch_bounds__(256) scales_kernel(const Params p, uint8_t* __restrict__ sfw, uint8_t* __restrict__ sfx, int tiles_w, int groups) {
    pdl_launch_dependents();
    pdl_wait();
    const int pairs = (p.num + 1) / 2;                    // a thread takes two stages: 16 scales of four rows
    const int units = (tiles_w + p.tiles_t * groups) * pairs;
    const int lane = threadIdx.x & 31;
    for (int u = blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += gridDim.x * 8) {
        const int unit = u / pairs, pair = u - unit * pairs;
        const bool of_w = unit < tiles_w;
        const int tt = (unit - tiles_w) / groups, group = (unit - tiles_w) - tt * groups;
        const uint8_t* base = of_w ? p.scales : p.a_scales;
        const uint8_t* end = base + (long long)(of_w ? p.w_rows : p.e.M) * p.blocks;
        const int b = pair * 16, n = p.blocks - b;
        uint32_t v[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = q * 32 + lane;
            const int row = of_w ? tile_row(p, unit, r) : min(tt * p.bn + group * 128 + r, p.e.M - 1);
            const uint8_t* src = base + (long long)row * p.blocks + b;
            if (n >= 16 && ((uintptr_t)src & 15) == 0) {
                const uint4 w = __ldg((const uint4*)src);
                v[q][0] = w.x; v[q][1] = w.y; v[q][2] = w.z; v[q][3] = w.w;
            } else {
                const uint2 lo = load8(src, base, end, n), hi = load8(src + 8, base, end, n - 8);
                v[q][0] = lo.x; v[q][1] = lo.y; v[q][2] = hi.x; v[q][3] = hi.y;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {                     // atoms of the two stages
            const int stage = pair * 2 + (j >> 1);
            if (stage >= p.num) break;
            uint8_t* at = of_w ? sfw + ((long long)unit * p.num + stage) * SFW_BYTES + (j & 1) * SF_ATOM
                               : sfx + (((long long)tt * p.num + stage) * 2 + (j & 1)) * groups * SF_ATOM + group * SF_ATOM;
            *(uint4*)(at + lane * 16) = make_uint4(v[0][j], v[1][j], v[2][j], v[3][j]);
        }
    }
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// An atom of scales from shared memory (32 rows of 16 bytes, groups of eight rows 128 bytes apart) to four columns of all four quarters.
__device__ __forceinline__ void copy_atom(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ uint64_t atom_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

__global__ void __launch_bounds__(THREADS4, 1)
gemm4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p, const uint8_t* __restrict__ sfw,
             const uint8_t* __restrict__ sfx, int groups) {
    static_assert(2 * MAX_BN + STAGES4 * SF_COLS <= 512, "tensor memory");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sSF = smem + STAGES4 * STAGE4_BYTES;         // [STAGES4][W's two atoms, the activations' two times `groups`]
    __shared__ uint64_t full[STAGES4], empty[STAGES4];
    __shared__ Rings d;
    __shared__ uint32_t tmem_base_smem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int num = p.num;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES4; ++i) { mbar_init(&full[i], 2); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&d.full[i], 2); mbar_init(&d.empty[i], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_x) : "memory");
    }
    pdl_wait();
    if (warp == 3) { tmem_alloc(&tmem_base_smem, 512u); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    constexpr uint32_t tmem_d = 0u, tmem_sf = 2 * MAX_BN;            // the whole of tensor memory is this CTA's
    bool ok = tmem_base_smem == 0u;                       // never anything else
    if (!ok) {
        if (threadIdx.x == 0) atomicExch(p.err, 90);
    } else if (warp == 0 || warp == 2) {
        // W's share of a stage and the activations', a thread each: a copy costs its thread about 100 cycles.
        if (lane == 0) {
            Ring<STAGES4> r;
            int n = 0;
            const uint32_t x_scales = (uint32_t)(2 * groups * SF_ATOM);
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
                const int tw = tile / p.tiles_t, tt = tile - tw * p.tiles_t;
                for (int i = 0; i < num; ++i, ++n) {
                    if (n >= STAGES4) { ok = mbar_wait(&empty[r.slot], r.pass ^ 1u, p.err, 111); if (!ok) break; }
                    uint8_t* at = smem + r.slot * STAGE4_BYTES;
                    uint8_t* sf = sSF + r.slot * (SFW_BYTES + SFX_BYTES);
                    if (warp == 0) {
                        mbar_expect_tx(&full[r.slot], (uint32_t)(CODE_BYTES + SFW_BYTES));
                        load_codes(p, at, &map_w, &full[r.slot], i * (CODE_K / 2), tw);
                        bulk_load(sf, sfw + ((long long)tw * num + i) * SFW_BYTES, SFW_BYTES, &full[r.slot]);
                    } else {
                        mbar_expect_tx(&full[r.slot], (uint32_t)(p.bn * (CODE_K / 2)) + x_scales);
                        tma_load_2d(at + CODE_BYTES, &map_x, &full[r.slot], i * (CODE_K / 2), tt * p.bn);
                        bulk_load(sf + SFW_BYTES, sfx + ((long long)tt * num + i) * x_scales, x_scales, &full[r.slot]);
                    }
                    r.next();
                }
            }
        }
        __syncwarp();
    } else if (warp < 4) {
        // Copies of scales and MMAs are carried out in the order in which they are issued.
        const int who = warp == 1 ? 0 : 1;
        const uint32_t idesc0 = idesc4(p.bn, 0), idesc2 = idesc4(p.bn, 2);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(smem)), sfdesc0 = atom_desc(smem_u32(sSF));
        const int total = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * num;
        int i = 0, it = 0;
        Ring<STAGES4> r;
        for (int n = 0; n < total; ++n) {
            if ((n & 1) == who) {
                if (ok && it >= 2 && i < 2) ok = mbar_wait(&d.empty[it & 1], (uint32_t)((it >> 1) - 1) & 1u, p.err, 112);
                ok = ok && mbar_wait(&full[r.slot], r.pass, p.err, 113);
                ok = __all_sync(0xffffffffu, ok);
                if (n) await_turn(who);
                tc_fence_after();
                const uint64_t adesc = desc0 + (uint64_t)(r.slot * (STAGE4_BYTES >> 4)), bdesc = adesc + (uint64_t)(CODE_BYTES >> 4);
                const uint64_t sfdesc = sfdesc0 + (uint64_t)(r.slot * ((SFW_BYTES + SFX_BYTES) >> 4));
                const uint32_t sf = tmem_sf + (uint32_t)(r.slot * SF_COLS), acc = tmem_d + (it & 1 ? MAX_BN : 0);
                if (ok && elected()) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {         // 128 columns of K
                        copy_atom(sf + 4u * k, sfdesc + (uint64_t)(k * (SF_ATOM >> 4)));
                        copy_atom(sf + 8u + 8u * k, sfdesc + (uint64_t)((SFW_BYTES + k * groups * SF_ATOM) >> 4));
                        if (groups == 2) copy_atom(sf + 12u + 8u * k, sfdesc + (uint64_t)((SFW_BYTES + (2 * k + 1) * SF_ATOM) >> 4));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)           // 64 columns of K = 32 bytes = 2 units of the address field
                        umma_mxf4(acc, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), k & 1 ? idesc2 : idesc0, sf + 4u * (k >> 1),
                                  sf + 8u + 8u * (k >> 1), (i > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&empty[r.slot]);
                    if (i >= num - 2) umma_commit(&d.full[it & 1]);
                    if (num == 1) umma_commit(&d.full[it & 1]);
                }
                __syncwarp();
                if (n + 1 < total) hand_on(who);
            }
            r.next();
            if (++i == num) { i = 0; ++it; }
        }
    } else if (warp >= 4) {
        ok = epilogue<2>(p, d, tmem_d, MAX_BN, (warp - 4) >> 2, [](int) { return 1.f; });
    }
    teardown(ok, tmem_base_smem, warp);
}

// ---- host -----------------------------------------------------------------------------------------
int g_forced_bn = 0;

// W's codes: rows in boxes of a tile's; gated, as [features / 8][gate, up][8 rows], so that a box is the tile's eight times eight gate rows and their up
// rows in turn (a box for every eight rows cost a thread more than the stage's MMAs took).  Features beside a multiple of eight: eight rows a box.
bool map_w(CUtensorMap* out, const void* codes, Params& p) {
    const int bytes = p.blocks * 16;
    p.one_box = 0;
    if (!p.e.gated) return map_bytes(out, codes, p.w_rows, bytes, TILE_W);
    if (p.e.N % 8 == 0) {
        EncodeTiledFn fn = encode_fn();
        if (!fn) return false;
        cuuint64_t dims[4] = {(cuuint64_t)bytes, 8u, 2u, (cuuint64_t)p.e.N / 8};
        cuuint64_t strides[3] = {(cuuint64_t)bytes, (cuuint64_t)bytes * p.e.N, (cuuint64_t)bytes * 8};
        cuuint32_t box[4] = {128u, 8u, 2u, 8u};
        cuuint32_t estr[4] = {1, 1, 1, 1};
        if (fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS) {
            p.one_box = 1;
            return true;
        }
    }
    return map_bytes(out, codes, p.w_rows, bytes, 8);
}

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

}  // namespace

// What a call would take, in ns (see the function of the same kind in gemm_mxfp4.cu): rounds of tiles, each its stages, whose time grows with the tile's
// tokens only in part.
TNX_EXPORT long long tnx_gemm_mxfp4_tiles_estimate(int M, int N, int K, int gated, int quantized, int n_sms) {
    Params p;
    p.e.M = M;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    plan(p, n_sms, tiles_w, quantized ? 430 : 360);
    const long long rounds = ((long long)p.tiles + n_sms - 1) / n_sms;
    return quantized ? rounds * ((K + CODE_K - 1) / CODE_K) * (300 + p.bn * 7 / 10) + 6500 : rounds * ((K + 127) / 128) * (500 + p.bn * 14 / 10) + 5000;
}

// For tests: the tokens of a tile (a multiple of 16 from 64 to 192) whatever the sizes (0: the plan's own).
TNX_EXPORT int tnx_gemm_mxfp4_tiles_force(int bn) {
    if (bn && (bn < 64 || bn > MAX_BN || bn % 16)) return TNX_ERR_BAD_ARG;
    g_forced_bn = bn;
    return 0;
}

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
    plan(p, n_sms, tiles_w, 360);
    CUtensorMap mw, mx;
    if (!map_w(&mw, codes, p) || !map_h16(&mx, a, M, K, lda, p.bn)) return TNX_ERR_UNSUPPORTED;
    static TnxSmemLimit limit;
    const int r = limit.allow(gemm16_kernel, SMEM16);
    if (r) return r;
    return tnx_launch_ex(1, gemm16_kernel, dim3(p.tiles < n_sms ? p.tiles : n_sms), dim3(THREADS16), SMEM16, stream, mw, mx, p);
}

// 4-bit activations: codes [M][blocks * 16] (16-byte aligned) and scales [M][blocks]; scratch: 16-byte aligned, for every 256 columns of K 1,024 bytes
// for 128 rows of W and 2,048 for 64 tokens.
TNX_EXPORT int tnx_gemm_mxfp4_tiles_4(const void* a, const void* a_scales, const void* codes, const void* scales, const float* bias, const float* residual,
                                      void* out, int out_h16, long long ldc, int M, int N, int K, int act, int gated, void* scratch, int n_sms, int* err,
                                      cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0 || ((uintptr_t)scratch & 15)) return TNX_ERR_BAD_ARG;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    if (((uintptr_t)a & 15) || ((uintptr_t)codes & 15) || (long long)tiles_w * ((M + 63) / 64) > 0x3FFFFFFF) return TNX_ERR_UNSUPPORTED;
    Params p;
    fill_epilogue(p.e, bias, residual, out, out_h16, ldc, M, N, act, gated);
    p.scales = (const uint8_t*)scales; p.a_scales = (const uint8_t*)a_scales; p.err = err;
    p.w_rows = gated ? 2 * N : N; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK; p.num = (K + CODE_K - 1) / CODE_K;
    plan(p, n_sms, tiles_w, 430);
    CUtensorMap mw, mx;
    if (!map_w(&mw, codes, p) || !map_bytes(&mx, a, M, p.blocks * 16, p.bn)) return TNX_ERR_UNSUPPORTED;
    static TnxSmemLimit limit;
    int r = limit.allow(gemm4_kernel, SMEM4);
    if (r) return r;
    const int groups = p.bn > 128 ? 2 : 1;
    uint8_t* sfw = (uint8_t*)scratch;
    uint8_t* sfx = sfw + (long long)tiles_w * p.num * SFW_BYTES;
    const long long units = (long long)(tiles_w + p.tiles_t * groups) * ((p.num + 1) / 2), blocks = (units + 7) / 8, most = (long long)n_sms * 8;
    r = tnx_launch_ex(1, scales_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, p, sfw, sfx, tiles_w, groups);
    if (r) return r;
    return tnx_launch_ex(1, gemm4_kernel, dim3(p.tiles < n_sms ? p.tiles : n_sms), dim3(THREADS4), SMEM4, stream, mw, mx, p, (const uint8_t*)sfw,
                         (const uint8_t*)sfx, groups);
}

// The same with the parameters in one array (the stream last): a call through ctypes costs 0.1 us a parameter.
TNX_EXPORT int tnx_gemm_mxfp4_tiles_16_packed(const long long* v) {
    return tnx_gemm_mxfp4_tiles_16((const void*)v[0], (long long)v[1], (const void*)v[2], (const void*)v[3], (const float*)v[4], (const float*)v[5],
                                   (void*)v[6], (int)v[7], (long long)v[8], (int)v[9], (int)v[10], (int)v[11], (int)v[12], (int)v[13], (int)v[14],
                                   (int*)v[15], (cudaStream_t)v[16]);
}
TNX_EXPORT int tnx_gemm_mxfp4_tiles_4_packed(const long long* v) {
    return tnx_gemm_mxfp4_tiles_4((const void*)v[0], (const void*)v[1], (const void*)v[2], (const void*)v[3], (const float*)v[4], (const float*)v[5],
                                  (void*)v[6], (int)v[7], (long long)v[8], (int)v[9], (int)v[10], (int)v[11], (int)v[12], (int)v[13], (void*)v[14],
                                  (int)v[15], (int*)v[16], (cudaStream_t)v[17]);
}
