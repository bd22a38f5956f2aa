// Products with a 4-bit matrix on the 5th-generation tensor cores.
//
//   out[t, n] = act( sum_k a[t, k] W[n, k] + bias[n] ) + residual[t, n]          W: microscaled 4 bits (mxfp4.cuh), 32-bit sums
//   gated:  out[t, f] = act( sum_k a[t, k] W[f, k] + bias[f] ) * ( sum_k a[t, k] W[F + f, k] + bias[F + f] )
//
// One CTA computes a tile of 128 rows of W (gated: 64 gate rows and the 64 up rows that go with them) by BN tokens.  W's rows are the 128
// lanes of the accumulator, the tokens its columns, so that a step of few tokens pads tokens to 16 and streams W once.  K may be split
// over the CTAs of a cluster.
//
// gemm16 (16-bit activations): W's codes come through TMA into shared memory, 256 columns of K a box; sixteen warps turn them into 16-bit
// values and put those into tensor memory, whence the MMAs take them as their A operand; activations come through TMA.  That turning is what
// bounds it, 0.75 us a box, beside 5 us a CTA has before its first box and behind its last: 16 tokens by 16,384 x 4,096 17 us (float16) and 20.5
// (bfloat16, whose values take more instructions), 14.7 and 13.4 without it, 13 and 11.4 also without MMAs; 13 by 5,120 x 20,480 27.5 and 31.5
// (2 and 1.8 TB/s), 128 by 2,048 x 8,192 15.  (Two warps that issue the MMAs in turn, as in gemm_mxfp4_tiles.cu, changed nothing here.)
//
// gemm4 (activations in 4 bits too): both operands' codes come through TMA, 256 columns of K a stage, and are multiplied as they are
// (tcgen05.mma kind::mxf4, a scale for 32 columns of K).  The MMAs read scales from tensor memory, where lane l of every quarter holds the
// scales of rows l, 32 + l, 64 + l ... in neighbouring columns, four blocks of K a column: eight warps load them row by row, exchange
// them through shared memory and store them there.  A stage takes 0.3 us, which the scales' way bounds: 24 tokens by 16,384 x 4,096 9.8 us, 32 by
// 4,096 x 4,096 7.
#include <atomic>

#include "gemm_mxfp4.cuh"

namespace {

constexpr int THREADS4 = 384;                // gemm4: warp 0: TMA, warp 1: MMAs, warps 4..11: scales, then sums
constexpr int GROUPS16 = 4;                  // gemm16: groups of four warps that make values
constexpr int THREADS16 = 128 + 128 * GROUPS16;      // warp 0: activations' TMA, warp 1: MMAs, warp 2: codes' TMA, warps 4..: values, then sums
constexpr int ROW_LD = TILE_W + 4;           // floats a token of the staged sums

struct Params {
    Epilogue e;
    const uint8_t* scales;
    const uint8_t* a_scales;                 // gemm4
    int tiles_t;                             // tiles of tokens: blockIdx.x counts them within those of W, of which there may be more than a grid's other axes hold
    int w_rows, blocks;                      // rows of W and scales a row
    int num_kb, boxes_per_split;             // K in stages; boxes of codes a CTA of the cluster takes
    int splits;
    int* err;
};

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t map_to_cta(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
    float4 f;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(a) : "memory");
    return f;
}
// The sums of a tile lie as [token][128 + 4 floats] at `sums` in the shared memory of every CTA of the cluster; this CTA writes every
// splits-th token.  A warp takes a token (gated: two), a lane four neighbouring features; partial sums are added in the order of the CTAs.
template <bool SPLIT, int THREADS>
__device__ __forceinline__ void write_tile(const Epilogue& e, uint32_t sums, int splits, int row0, int token0, int tokens) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = SPLIT ? (int)cta_rank() : 0;
    if (!SPLIT) splits = 1;
    auto load = [&](int t, int f) {
        const uint32_t a = sums + (uint32_t)(t * ROW_LD + f) * 4u;
        if (!SPLIT) {
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
            return v;
        }
        float4 v = ld_cluster4(map_to_cta(a, 0));
        for (int s = 1; s < splits; ++s) {
            const float4 u = ld_cluster4(map_to_cta(a, (uint32_t)s));
            v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        return v;
    };
    const int f = e.gated ? 4 * (lane & 15) : 4 * lane;              // this lane's features within the tile
    const int n = (e.gated ? row0 / 2 : row0) + f;
    if (n >= e.N) return;
    const bool vec = e.vec && n + 3 < e.N;
    float b[4] = {0.f, 0.f, 0.f, 0.f}, bu[4] = {0.f, 0.f, 0.f, 0.f};
    if (e.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < e.N) { b[j] = __ldg(e.bias + n + j); if (e.gated) bu[j] = __ldg(e.bias + e.N + n + j); }
    }
    const int step = (THREADS / 32) * (e.gated ? 2 : 1);
    for (int i = e.gated ? 2 * warp + (lane >> 4) : warp; i * splits + rank < tokens; i += step) {
        const int t = i * splits + rank;
        const long long o = (long long)(token0 + t) * e.ldc + n;
        float res[4] = {0.f, 0.f, 0.f, 0.f};
        if (e.residual) {
            if (vec) { const float4 r = __ldcg((const float4*)(e.residual + o)); res[0] = r.x; res[1] = r.y; res[2] = r.z; res[3] = r.w; }
            else
                for (int j = 0; j < 4; ++j) if (n + j < e.N) res[j] = __ldcg(e.residual + o + j);
        }
        const float4 s = load(t, f);
        float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = e.out_h16 ? activate(v[j] + b[j], e.act) : mx_activation(v[j] + b[j], e.act);
        if (e.gated) {
            const float4 u = load(t, 64 + f);
            v[0] *= u.x + bu[0]; v[1] *= u.y + bu[1]; v[2] *= u.z + bu[2]; v[3] *= u.w + bu[3];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += res[j];
        if (vec) {
            if (e.out_h16) {
                const h16x2 h0 = floats_to_h16x2(v[0], v[1]), h1 = floats_to_h16x2(v[2], v[3]);
                *(uint2*)((h16*)e.out + o) = make_uint2(*(const uint32_t*)&h0, *(const uint32_t*)&h1);
            } else *(float4*)((float*)e.out + o) = make_float4(v[0], v[1], v[2], v[3]);
        } else
            for (int j = 0; j < 4; ++j)
                if (n + j < e.N) { if (e.out_h16) ((h16*)e.out)[o + j] = float_to_h16(v[j]); else ((float*)e.out)[o + j] = v[j]; }
    }
}

// Row `r` of a tile (gated: 64 gate rows, then their 64 up rows) in W; rows behind the last count as the last one (their sums are not written).
__device__ __forceinline__ int tile_row(const Epilogue& e, int row0, int r, int w_rows) {
    const int row = !e.gated ? row0 + r : r < 64 ? row0 / 2 + r : e.N + row0 / 2 + r - 64;
    return row < w_rows ? row : w_rows - 1;
}

// A warp's share of the sums, from tensor memory to shared memory: the stages are idle once the last MMA is done.
template <int BN, int GROUPS, int ACCS = 1>
__device__ __forceinline__ void stage_sums(uint8_t* smem, uint32_t tmem_d, int quad, int group, int lane, bool ok, bool scaled = false, float factor = 1.f) {
    float* sums = (float*)smem + quad * 32 + lane;
    constexpr int COLS = BN < 32 * GROUPS ? 16 : 32;
#pragma unroll 1
    for (int c = group * COLS; c < BN; c += GROUPS * COLS) {
        uint32_t v[32];
        if (ok) {
            const uint32_t at = tmem_d + ((uint32_t)(quad * 32) << 16) + (uint32_t)c;
            if (COLS == 32) tmem_ld32(at, v); else tmem_ld16(at, v);
            tmem_ld_wait();
#pragma unroll
            for (int a = 1; a < ACCS; ++a) {
                uint32_t u[32];
                if (COLS == 32) tmem_ld32(at + (uint32_t)(a * BN), u); else tmem_ld16(at + (uint32_t)(a * BN), u);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < COLS; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
            }
        }
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
            float f = ok ? __uint_as_float(v[j]) : 0.f;                            // defined even if a wait ran out
#ifdef TNX_F16
            if (scaled) f = f * (1.f / (float)(1 << MX_F16_TOP)) * factor;
#endif
            sums[(c + j) * ROW_LD] = f;
        }
    }
}

// What all warps do behind the sums: wait for the staged tile (of all CTAs of the cluster), write it.
template <int BN, int THREADS>
__device__ __forceinline__ void finish_tile(const Params& p, uint8_t* smem, bool ok, int row0, int token0) {
    if (!ok) {
        // A wait ran out: give copies in flight time to land before the shared memory is used otherwise.
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before();
    if (p.splits > 1) {
        cluster_sync();
        write_tile<true, THREADS>(p.e, smem_u32(smem), p.splits, row0, token0, min(BN, p.e.M - token0));
        __syncwarp();
        cluster_sync();                                   // no CTA leaves while its sums may still be read
    } else {
        __syncthreads();
        write_tile<false, THREADS>(p.e, smem_u32(smem), 1, row0, token0, min(BN, p.e.M - token0));
        __syncthreads();
    }
}

// Tensor memory is asked for behind the wait for the preceding kernel and before the next one may start, and what else an SM can hold beside a CTA
// leaves it enough: whoever waits for tensor memory then waits for CTAs that end by themselves.  (A CTA of the next kernel that held some while it
// waited for this one, or CTAs of two kernels on two streams whose clusters each hold what the other's want, would never end.)  gemm16 takes all of
// it, so a CTA of a cluster takes the SM's shared memory too; gemm4's CTAs take a quarter and half of the shared memory, or (128 tokens) half.

// A stage is a box of codes: 256 columns of K, 16 MMAs.  (With 64 columns a stage, the waits and commits of the MMAs' warp, 250 to 300 cycles a stage
// whatever it multiplies, were half of the kernel: one to 64 tokens by 16,384 x 4,096 22 us.)
template <int BN> __host__ __device__ constexpr int x_stage_bytes() { return BN * CODE_K * 2; }
template <int BN, int STAGES, int BOXES> __host__ __device__ constexpr int gemm16_smem() { return BOXES * CODE_BYTES + STAGES * x_stage_bytes<BN>() + 1024; }
template <int BN> __host__ __device__ constexpr int gemm16_accs() { return BN <= 32 ? 4 : BN <= 64 ? 2 : 1; }       // shorter chains of additions where there is room

// BN tokens; STAGES: stages of activations and values in flight; BOXES: boxes of codes.
template <int BN, int STAGES, int BOXES>
__global__ void __launch_bounds__(THREADS16, 1)
gemm16_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
    constexpr int X_BYTES = x_stage_bytes<BN>(), ACCS = gemm16_accs<BN>(), PARTS = CODE_K / KB, A_COLS = CODE_K / 2;
    static_assert(ACCS * BN + STAGES * A_COLS <= 512, "tensor memory");
    static_assert(GROUPS16 == PARTS, "a group of warps for every K block of a box");
    static_assert(BN * ROW_LD * 4 <= BOXES * CODE_BYTES + STAGES * X_BYTES, "the staged sums take the place of the stages");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sW = smem;                                   // [BOXES]
    uint8_t* sX = smem + BOXES * CODE_BYTES;              // [STAGES][K blocks]
    __shared__ uint64_t w_full[BOXES], w_empty[BOXES], full[STAGES], empty[STAGES], done;
    __shared__ uint32_t tmem_base_smem;
#ifdef TNX_F16
    __shared__ int row_ref[TILE_W];
#endif

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_w = (int)blockIdx.x / p.tiles_t, token0 = ((int)blockIdx.x - tile_w * p.tiles_t) * BN, row0 = tile_w * TILE_W;
    const int box0 = (int)blockIdx.z * p.boxes_per_split;
    const int kb0 = box0 * PARTS;
    const int num_kb = min(p.num_kb - kb0, p.boxes_per_split * PARTS);               // at least one
    const int num_boxes = (num_kb + PARTS - 1) / PARTS;

    if (threadIdx.x == 0) {
        for (int i = 0; i < BOXES; ++i) { mbar_init(&w_full[i], 1); mbar_init(&w_empty[i], 4 * GROUPS16); }
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1 + 4 * GROUPS16); mbar_init(&empty[i], 1); }         // full: activations and all warps' values
        mbar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_x) : "memory");
    }
    pdl_wait();                                           // codes, scales and activations may be the preceding kernel's
    if (warp == 1) { tmem_alloc(&tmem_base_smem, 512u); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();                              // see Tensor memory, above
    const uint32_t tmem_d = tmem_base_smem, tmem_a = tmem_d + ACCS * BN;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < num_boxes && ok; ++i) {
                const int s = i % STAGES, parts = min(PARTS, num_kb - i * PARTS);
                if (i >= STAGES) { ok = mbar_wait(&empty[s], (uint32_t)(i / STAGES - 1) & 1u, p.err, 62); if (!ok) break; }
                mbar_expect_tx(&full[s], (uint32_t)(parts * BN * KB * 2));
                for (int j = 0; j < parts; ++j)
                    tma_load_2d(sX + s * X_BYTES + j * (BN * KB * 2), &map_x, &full[s], (kb0 + i * PARTS + j) * KB, token0);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        if (lane == 0) {
            const int g0 = p.e.gated ? row0 / 2 : row0, g1 = p.e.gated ? p.e.N + row0 / 2 : row0 + 64;
            for (int i = 0; i < num_boxes && ok; ++i) {
                const int s = i % BOXES;
                if (i >= BOXES) { ok = mbar_wait(&w_empty[s], (uint32_t)(i / BOXES - 1) & 1u, p.err, 61); if (!ok) break; }
                mbar_expect_tx(&w_full[s], CODE_BYTES);
                const int x = (box0 + i) * (CODE_K / 2);
                tma_load_2d(sW + s * CODE_BYTES, &map_w, &w_full[s], x, g0);
                tma_load_2d(sW + s * CODE_BYTES + CODE_BYTES / 2, &map_w, &w_full[s], x, g1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc16(BN);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(sX));
        Ring<STAGES> r;
        for (int i = 0; i < num_boxes && ok; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[r.slot], r.pass, p.err, 63));
            if (!ok) break;
            tc_fence_after();
            const int parts = min(PARTS, num_kb - i * PARTS);
            const uint64_t bdesc = desc0 + (uint64_t)(r.slot * (X_BYTES >> 4));
            const uint32_t a = tmem_a + (uint32_t)(r.slot * A_COLS);
            if (elected()) {
#pragma unroll
                for (int j = 0; j < PARTS; ++j) {
                    if (j >= parts) break;
#pragma unroll
                    for (int k = 0; k < KB / 16; ++k)
                        umma_a_tmem(tmem_d + (uint32_t)(k % ACCS * BN), a + (uint32_t)(32 * j + 8 * k), bdesc + (uint64_t)(j * (BN * KB * 2 >> 4) + 2 * k), idesc,
                                    (i > 0 || j > 0 || k >= ACCS) ? 1u : 0u);
                }
                umma_commit(&empty[r.slot]);
                if (i == num_boxes - 1) umma_commit(&done);
            }
            __syncwarp();
            r.next();
        }
    } else if (warp >= 4) {
        // Values: warp w fills the lanes of quarter w % 4 (which its tensor memory accesses are confined to), each group of four
        // warps takes one of a box's four K blocks.  A thread owns a row.
        const int quad = warp & 3, group = (warp - 4) >> 2, r = quad * 32 + lane;
        const uint8_t* sc = p.scales + (long long)tile_row(p.e, row0, r, p.w_rows) * p.blocks;
        const int blk0 = box0 * (CODE_K / MX_BLOCK), blk_end = min(p.blocks, blk0 + num_kb * 2);
        const bool even = p.blocks % 2 == 0 && ((uintptr_t)p.scales & 1) == 0;
        auto load_scales = [&](int box) -> uint32_t {     // the two scales of this group's K block of a box
            const int b = blk0 + box * 8 + 2 * group;
            if (b >= blk_end) return 0u;
            if (even) return __ldg((const uint16_t*)(sc + b));
            return (uint32_t)__ldg(sc + b) | (b + 1 < p.blocks ? (uint32_t)__ldg(sc + b + 1) << 8 : 0u);
        };
        // Asked for four boxes ahead: a trip to memory takes longer than a box.  (The loop is unrolled so that a register waits for its load
        // where the scale is used: handing the values on would wait for the newest.)
        uint32_t ahead[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ahead[j] = load_scales(j);
        int ref = 0;
#ifdef TNX_F16
        // the largest scale of every row over this CTA's share of K, which becomes a factor of the row's sums
        {
            const bool wide = p.blocks % 8 == 0 && ((uintptr_t)p.scales & 7) == 0;
            const int n = blk_end - blk0, t = (warp - 4) * 32 + lane;
            static_assert(2 * 16 * GROUPS16 == TILE_W, "eight threads a row, two rows each");
            const uint8_t* q[2];
            int m[2] = {0, 0};
#pragma unroll
            for (int h = 0; h < 2; ++h) q[h] = p.scales + (long long)tile_row(p.e, row0, (t >> 3) + h * (TILE_W / 2), p.w_rows) * p.blocks + blk0;
            if (wide) {
#pragma unroll 4
                for (int j = (t & 7) * 8; j < n; j += 64) {
                    uint2 v[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) v[h] = __ldg((const uint2*)(q[h] + j));
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k = 0; k < 8; ++k) { const int E = (int)(((k < 4 ? v[h].x : v[h].y) >> (8 * (k & 3))) & 255u); if (E < 255) m[h] = max(m[h], E); }
                }
            } else {
#pragma unroll 4
                for (int j = t & 7; j < n; j += 8) {
                    int E[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) E[h] = __ldg(q[h] + j);
#pragma unroll
                    for (int h = 0; h < 2; ++h) if (E[h] < 255) m[h] = max(m[h], E[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                m[h] = max(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
                m[h] = max(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
                m[h] = max(m[h], __shfl_xor_sync(0xffffffffu, m[h], 4));
                if ((t & 7) == 0) row_ref[(t >> 3) + h * (TILE_W / 2)] = m[h];
            }
            asm volatile("bar.sync 1, %0;" ::"n"(128 * GROUPS16) : "memory");
            ref = row_ref[r];
        }
#endif
        for (int box4 = 0; box4 < num_boxes && ok; box4 += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int box = box4 + u, ws = box % BOXES, s = box % STAGES;
                if (box >= num_boxes || !ok) break;
                const uint32_t two = ahead[u];
                ahead[u] = load_scales(box + 4);
                ok = __all_sync(0xffffffffu, mbar_wait(&w_full[ws], (uint32_t)(box / BOXES) & 1u, p.err, 65));
                if (!ok) break;
                const bool has = box * PARTS + group < num_kb;       // the last box may end before this group's K block
                const uint32_t row_addr = smem_u32(sW + ws * CODE_BYTES) + (uint32_t)r * 128u;
                uint4 q[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t at = row_addr + ((uint32_t)((2 * group + c) ^ (r & 7)) << 4);
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[c].x), "=r"(q[c].y), "=r"(q[c].z), "=r"(q[c].w) : "r"(at) : "memory");
                }
                uint32_t v[32];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const MxValues t((two >> (8 * c)) & 255u, ref);
                    t.decode8(q[c].x, &v[16 * c]);
                    t.decode8(q[c].y, &v[16 * c + 4]);
                    t.decode8(q[c].z, &v[16 * c + 8]);
                    t.decode8(q[c].w, &v[16 * c + 12]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&w_empty[ws]);                             // this warp has read its share of the box
                if (box >= STAGES) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (uint32_t)(box / STAGES - 1) & 1u, p.err, 66));
                    if (!ok) break;
                    tc_fence_after();
                }
                if (has) {
                    tmem_st32(tmem_a + (uint32_t)(s * A_COLS + group * 32) + ((uint32_t)(quad * 32) << 16), v);
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
            }
        }
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&done, 0, p.err, 67));
        tc_fence_after();
#ifdef TNX_F16
        stage_sums<BN, GROUPS16, ACCS>(smem, tmem_d, quad, group, lane, ok, true, mx_scale((uint32_t)ref));
#else
        stage_sums<BN, GROUPS16, ACCS>(smem, tmem_d, quad, group, lane, ok);
#endif
    }
    finish_tile<BN, THREADS16>(p, smem, ok, row0, token0);
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base_smem, 512u); }
}

// ---- both operands in 4 bits -----------------------------------------------------------------------
// A stage's scales in tensor memory: two atoms (four blocks of K) of four columns for W, two for the activations.
constexpr int SF_COLS = 16;
template <int BN> __host__ __device__ constexpr int sf_cols_x() { return BN < 32 ? 1 : BN / 32; }         // columns of an atom with tokens in them
template <int BN, int STAGES> __host__ __device__ constexpr int gemm4_smem() { return STAGES * (CODE_BYTES + BN * CODE_K / 2) + 1024; }
template <int BN, int STAGES> __host__ __device__ constexpr uint32_t gemm4_tmem() {
    return BN + STAGES * SF_COLS <= 128 ? 128u : BN + STAGES * SF_COLS <= 256 ? 256u : 512u;
}

__device__ __forceinline__ void group_sync(int group) {
    if (group) asm volatile("bar.sync 2, 128;" ::: "memory");
    else asm volatile("bar.sync 1, 128;" ::: "memory");
}

template <int BN, int STAGES, int CTAS>
__global__ void __launch_bounds__(THREADS4, CTAS)
gemm4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
    constexpr int STAGE_BYTES = CODE_BYTES + BN * CODE_K / 2;
    constexpr uint32_t TMEM_COLS = gemm4_tmem<BN, STAGES>();
    constexpr int XC = sf_cols_x<BN>();
    static_assert(BN * ROW_LD * 4 <= STAGES * STAGE_BYTES, "the staged sums take the place of the stages");
    static_assert(STAGES % 2 == 0, "two groups of warps fill the scales in turn");
    static_assert(BN <= 128, "a thread loads a row of the activations' scales");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[STAGES], sf_full[STAGES], empty[STAGES], done;
    __shared__ uint32_t tmem_base_smem;
    __shared__ uint32_t sf_smem[2][SF_COLS * 32];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_w = (int)blockIdx.x / p.tiles_t, token0 = ((int)blockIdx.x - tile_w * p.tiles_t) * BN, row0 = tile_w * TILE_W;
    const int st0 = (int)blockIdx.z * p.boxes_per_split;                           // stages of 256 columns
    const int num = min((p.blocks + 7) / 8 - st0, p.boxes_per_split);               // at least one

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&sf_full[i], 4); mbar_init(&empty[i], 1); }
        mbar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&map_x) : "memory");
    }
    pdl_wait();                                           // codes, scales and activations may be the preceding kernel's
    if (warp == 1) { tmem_alloc(&tmem_base_smem, TMEM_COLS); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();                              // see Tensor memory, above
    const uint32_t tmem_d = tmem_base_smem, tmem_sf = tmem_d + BN;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            const int g0 = p.e.gated ? row0 / 2 : row0, g1 = p.e.gated ? p.e.N + row0 / 2 : row0 + 64;
            for (int i = 0; i < num && ok; ++i) {
                const int s = i % STAGES;
                if (i >= STAGES) { ok = mbar_wait(&empty[s], (uint32_t)(i / STAGES - 1) & 1u, p.err, 71); if (!ok) break; }
                mbar_expect_tx(&full[s], STAGE_BYTES);
                uint8_t* at = smem + s * STAGE_BYTES;
                const int x = (st0 + i) * (CODE_K / 2);
                tma_load_2d(at, &map_w, &full[s], x, g0);
                tma_load_2d(at + CODE_BYTES / 2, &map_w, &full[s], x, g1);
                tma_load_2d(at + CODE_BYTES, &map_x, &full[s], x, token0);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint64_t desc0 = smem_desc_sw128(smem_u32(smem));
        Ring<STAGES> r;
        for (int i = 0; i < num && ok;) {
            int ready = min(ready_stages(full, r.slot, r.pass, STAGES, sf_full, r.slot, r.pass, STAGES), num - i);
            if (ready == 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&full[r.slot], r.pass, p.err, 72) && mbar_wait(&sf_full[r.slot], r.pass, p.err, 73));
                if (!ok) break;
                ready = 1;
            }
            tc_fence_after();
            for (; ready > 0; --ready, ++i) {
                const uint64_t adesc = desc0 + (uint64_t)(r.slot * (STAGE_BYTES >> 4)), bdesc = adesc + (uint64_t)(CODE_BYTES >> 4);
                const uint32_t sf = tmem_sf + (uint32_t)(r.slot * SF_COLS);
                if (elected()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)           // 64 columns of K = 32 bytes = 2 units of the address field
                        umma_mxf4(tmem_d, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc4(BN, (k & 1) * 2), sf + 4u * (k >> 1),
                                  sf + 8u + 4u * (k >> 1), (i > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&empty[r.slot]);
                    if (i == num - 1) umma_commit(&done);
                }
                __syncwarp();
                r.next();
            }
        }
    } else if (warp >= 4) {
        // Scales: two groups of four warps take stages in turn; a thread loads a row of W's and one of the activations', eight scales each,
        // three turns ahead (a trip to memory takes longer than a stage); then every warp stores all of them to the lanes of its quarter.
        const int quad = warp & 3, group = (warp - 4) >> 2, r = quad * 32 + lane;
        const uint8_t* w_end = p.scales + (long long)p.w_rows * p.blocks;
        const uint8_t* x_end = p.a_scales + (long long)p.e.M * p.blocks;
        const uint8_t* ws = p.scales + (long long)tile_row(p.e, row0, r, p.w_rows) * p.blocks;
        const int t = token0 + r < p.e.M ? token0 + r : p.e.M - 1;
        const uint8_t* xs = p.a_scales + (long long)t * p.blocks;
        struct Scales { uint2 w, x; };
        auto load = [&](int i) {
            Scales q;
            const int b = (st0 + i) * 8, n = i < num ? p.blocks - b : 0;
            q.w = load8(ws + b, p.scales, w_end, n);
            if (r < 32 * XC) q.x = load8(xs + b, p.a_scales, x_end, n);
            return q;
        };
        uint32_t* buf = sf_smem[group];
        Scales ahead[3] = {load(group), load(group + 2), load(group + 4)};
        for (int i0 = group; i0 < num; i0 += 6) {         // whole even if a wait ran out: the groups' warps meet at their barrier
#pragma unroll
          for (int u = 0; u < 3; ++u) {                   // (unrolled so that a register waits for its load where it is used)
            const int i = i0 + 2 * u;
            if (i >= num) break;
            const Scales now = ahead[u];
            ahead[u] = load(i + 6);
            buf[quad * 32 + lane] = now.w.x; buf[(4 + quad) * 32 + lane] = now.w.y;
            if (r < 32 * XC) { buf[(8 + quad) * 32 + lane] = now.x.x; buf[(12 + quad) * 32 + lane] = now.x.y; }
            group_sync(group);
            uint32_t v[SF_COLS];
#pragma unroll
            for (int c = 0; c < SF_COLS; ++c) v[c] = c < 8 || c % 4 < XC ? buf[c * 32 + lane] : 0u;
            const int s = i % STAGES;
            if (ok && i >= STAGES) {
                ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (uint32_t)(i / STAGES - 1) & 1u, p.err, 74));
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
                if (lane == 0) mbar_arrive(&sf_full[s]);
            }
            group_sync(group);                            // the buffer has been read by all four
          }
        }
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&done, 0, p.err, 75));
        tc_fence_after();
        stage_sums<BN, 2>(smem, tmem_d, quad, group, lane, ok);
    }
    finish_tile<BN, THREADS4>(p, smem, ok, row0, token0);
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base_smem, TMEM_COLS); }
}

// ---- host -----------------------------------------------------------------------------------------
// How many CTAs of a kernel the device holds at a time in clusters of S when an SM has one of them, asked for once a device and kernel.
struct Places {
    std::atomic<int> known[64][9];
    template <typename Kernel> int of(Kernel kernel, int threads, int smem, int S, int n_sms) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64) return n_sms;
        int n = known[dev][S].load();
        if (n) return n;
        if (S == 1) {
            n = n_sms;
        } else {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1, 1, S); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = S;
            cfg.attrs = attr; cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
            n = n < 1 ? n_sms / 2 : n * S;
        }
        known[dev][S].store(n);
        return n;
    }
};

int g_forced_splits = 0, g_forced_bn = 0;

// The split of K over a cluster's CTAs, any number up to eight that leaves none without work: rounds of CTAs, each its boxes of 256 columns and what
// it costs beside them, as much as `fixed` boxes; a part of a sum to be joined costs about one (13 float16 tokens by 5,120 x 20,480: 64 us unsplit,
// 35 in two, 28 in three, 42 in four, which need two rounds).  chain: the most columns of K that one accumulator should add up (0: any number): an
// addition cuts off what it shifts out, so what a sum loses grows with its chain.  Returns the estimate in boxes.
template <typename PlacesOf>
long long split(Params& p, int bn, int tiles_w, int fixed, int chain, PlacesOf places_of) {
    const int boxes = (p.blocks + CODE_K / MX_BLOCK - 1) / (CODE_K / MX_BLOCK);
    const long long tiles = (long long)tiles_w * ((p.e.M + bn - 1) / bn);
    int least = 1;
    while (chain && least < 8 && p.blocks * MX_BLOCK > chain * least) ++least;
    long long best = -1;
    p.splits = 1; p.boxes_per_split = boxes;
    for (int S = 1; S <= 8; ++S) {
        const int per = (boxes + S - 1) / S;
        if ((boxes + per - 1) / per != S) continue;
        if (g_forced_splits ? S != g_forced_splits : S < least && boxes >= least) continue;
        const int places = places_of(S);
        const long long rounds = (tiles * S + places - 1) / places, cost = rounds * (per + fixed) + S;
        if (best < 0 || cost < best) { best = cost; p.splits = S; p.boxes_per_split = per; }
    }
    return best < 0 ? boxes + fixed + 1 : best;
}

template <typename Kernel>
int launch(Kernel kernel, int threads, int smem, int bn, const CUtensorMap& mw, const CUtensorMap& mx, Params& p, int tiles_w, cudaStream_t stream) {
    p.tiles_t = (p.e.M + bn - 1) / bn;
    if ((long long)p.tiles_t * tiles_w > 0x7FFFFFFF) return TNX_ERR_UNSUPPORTED;
    const dim3 grid(p.tiles_t * tiles_w, 1, p.splits);
    if (p.splits > 1) return tnx_launch_cluster(1, dim3(1, 1, p.splits), kernel, grid, dim3(threads), smem, stream, mw, mx, p);
    return tnx_launch_ex(1, kernel, grid, dim3(threads), smem, stream, mw, mx, p);
}

constexpr int SMEM_ALONE = 220 * 1024, SMEM_HALF = 106 * 1024;        // beside them: nothing that uses tensor memory; one more
constexpr int FIXED16 = 8, FIXED4 = 20;      // what a CTA costs beside its boxes, in boxes

// cost: only the estimate is wanted, nothing is launched.
template <int BN, int STAGES, int BOXES>
int launch16(const void* a, long long lda, const void* codes, int K, Params& p, int tiles_w, int chain, int n_sms, cudaStream_t stream, long long* cost = nullptr) {
    static TnxSmemLimit limit;
    static Places places;
    auto kernel = gemm16_kernel<BN, STAGES, BOXES>;
    constexpr int SMEM = gemm16_smem<BN, STAGES, BOXES>();
    static_assert(SMEM <= SMEM_ALONE, "shared memory");
    const int r = limit.allow(kernel, SMEM_ALONE);
    if (r) return r;
    const long long boxes = split(p, BN, tiles_w, FIXED16, chain, [&](int S) { return places.of(kernel, THREADS16, SMEM_ALONE, S, n_sms); });
    if (cost) { *cost = boxes; return 0; }
    CUtensorMap mw, mx;
    if (!map_bytes(&mw, codes, p.w_rows, p.blocks * 16, 64) || !map_h16(&mx, a, p.e.M, K, lda, BN)) return TNX_ERR_UNSUPPORTED;
    return launch(kernel, THREADS16, p.splits > 1 ? SMEM_ALONE : SMEM, BN, mw, mx, p, tiles_w, stream);
}
template <int BN, int STAGES, int CTAS>
int launch4(const void* a, const void* codes, Params& p, int tiles_w, int n_sms, cudaStream_t stream, long long* cost = nullptr) {
    static TnxSmemLimit limit;
    static Places places;
    auto kernel = gemm4_kernel<BN, STAGES, CTAS>;
    constexpr int SMEM = CTAS == 2 ? SMEM_HALF : gemm4_smem<BN, STAGES>();
    static_assert(gemm4_smem<BN, STAGES>() <= SMEM, "shared memory");
    const int r = limit.allow(kernel, SMEM);
    if (r) return r;
    const long long boxes = split(p, BN, tiles_w, FIXED4, 0, [&](int S) { return CTAS * places.of(kernel, THREADS4, SMEM, S, n_sms); });
    if (cost) { *cost = boxes; return 0; }
    CUtensorMap mw, mx;
    if (!map_bytes(&mw, codes, p.w_rows, p.blocks * 16, 64) || !map_bytes(&mx, a, p.e.M, p.blocks * 16, BN)) return TNX_ERR_UNSUPPORTED;
    return launch(kernel, THREADS4, SMEM, BN, mw, mx, p, tiles_w, stream);
}

// Random operands, relative errors of 32-bit results: float16 3.8e-7 over chains of 4,096 columns, 1.2e-6 over 8,192, 5.5e-6 over 20,480; bfloat16, whose
// products have fewer bits, 0.8e-7, 2.2e-7 and 1e-6 to 2e-6.  With the limit, 100 bfloat16 tokens: 1.6e-7 over 20,480, 3.4e-7 over 40,960 where scales are alike,
// 2.3e-6 and 4.5e-6 where they spread over 2^16; beyond eight chains, 40,960 columns, more again (6e-7 and 7.2e-6 over 65,536).  Both operands in 4 bits: an
// addition for 64 columns; one accumulator's 0.7e-6 over 20,480 and 2.1e-6 over 65,536 (scales over 2^16; 0.5e-7 and 0.8e-7 over 2^8) need no limit.
constexpr int MX_CHAIN = 5120;

void fill(Params& p, const void* scales, const void* a_scales, const float* bias, const float* residual, void* out, int out_h16, long long ldc, int M, int N,
          int K, int act, int gated, int* err) {
    fill_epilogue(p.e, bias, residual, out, out_h16, ldc, M, N, act, gated);
    p.scales = (const uint8_t*)scales; p.a_scales = (const uint8_t*)a_scales;
    p.w_rows = gated ? 2 * N : N; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK; p.err = err;
    p.num_kb = (K + KB - 1) / KB;
}
int tile_tokens(int M) { return g_forced_bn ? g_forced_bn : M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128; }

}  // namespace

// What a call would take, in ns, for a choice between this file's kernels and gemm_mxfp4_tiles.cu's: rounds of CTAs, each its boxes of 256 columns and
// what a CTA costs beside them (fitted to more than 128 tokens, whose tiles are 128 wide; `quantized`: 4-bit activations).
TNX_EXPORT long long tnx_gemm_mxfp4_estimate(int M, int N, int K, int gated, int quantized, int out_h16, int n_sms) {
    Params p;
    p.e.M = M;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    long long boxes = 0;
    const int r = quantized ? launch4<128, 4, 1>(nullptr, nullptr, p, tiles_w, n_sms, nullptr, &boxes)
                            : launch16<128, 2, 4>(nullptr, 0, nullptr, K, p, tiles_w, out_h16 ? 0 : MX_CHAIN, n_sms, nullptr, &boxes);
    if (r) return 1ll << 60;
    // a box takes 650 (4-bit activations) or 1,150 ns; what a CTA costs beside them is 6.5 us, with 4-bit activations 0.3 more for every part of a sum
    const long long rounds = (boxes - p.splits) / (p.boxes_per_split + (quantized ? FIXED4 : FIXED16));
    return rounds * (p.boxes_per_split * (quantized ? 650ll : 1150ll) + 6500 + (quantized ? 300 * p.splits : 0));
}

// The most columns of K for whose 32-bit sums a tile's one accumulator is near enough (gemm_mxfp4_tiles.cu has one a tile).
TNX_EXPORT int tnx_gemm_mxfp4_chain() { return MX_CHAIN; }

// For tests: the tokens of a tile (16, 32, 64 or 128) and the split of K (1 to 8, where K allows it) whatever the sizes (0: the plan's own).
TNX_EXPORT int tnx_gemm_mxfp4_force(int bn, int splits) {
    if ((bn && bn != 16 && bn != 32 && bn != 64 && bn != 128) || splits < 0 || splits > 8) return TNX_ERR_BAD_ARG;
    g_forced_bn = bn; g_forced_splits = splits;
    return 0;
}

// 16-bit activations [M, K] (pitch lda, a multiple of 8 elements, 16-byte aligned) by codes [w_rows][blocks * 16] (16-byte aligned).
TNX_EXPORT int tnx_gemm_mxfp4_16(const void* a, long long lda, const void* codes, const void* scales, const float* bias, const float* residual, void* out,
                                 int out_h16, long long ldc, int M, int N, int K, int act, int gated, int n_sms, int* err, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0) return TNX_ERR_BAD_ARG;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    if (lda % 8 || ((uintptr_t)a & 15) || ((uintptr_t)codes & 15)) return TNX_ERR_UNSUPPORTED;
    Params p;
    fill(p, scales, nullptr, bias, residual, out, out_h16, ldc, M, N, K, act, gated, err);
    const int chain = out_h16 ? 0 : MX_CHAIN;
    switch (tile_tokens(M)) {
        case 16: return launch16<16, 3, 6>(a, lda, codes, K, p, tiles_w, 4 * chain, n_sms, stream);         // four accumulators share a sum
        case 32: return launch16<32, 3, 6>(a, lda, codes, K, p, tiles_w, 4 * chain, n_sms, stream);
        case 64: return launch16<64, 3, 6>(a, lda, codes, K, p, tiles_w, 2 * chain, n_sms, stream);
        default: return launch16<128, 2, 4>(a, lda, codes, K, p, tiles_w, chain, n_sms, stream);
    }
}

// 4-bit activations: codes [M][blocks * 16] (16-byte aligned) and scales [M][blocks].
TNX_EXPORT int tnx_gemm_mxfp4_4(const void* a, const void* a_scales, const void* codes, const void* scales, const float* bias, const float* residual, void* out,
                                int out_h16, long long ldc, int M, int N, int K, int act, int gated, int n_sms, int* err, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0) return TNX_ERR_BAD_ARG;
    const int tiles_w = gated ? (N + 63) / 64 : (N + TILE_W - 1) / TILE_W;
    if (((uintptr_t)a & 15) || ((uintptr_t)codes & 15)) return TNX_ERR_UNSUPPORTED;
    Params p;
    fill(p, scales, a_scales, bias, residual, out, out_h16, ldc, M, N, K, act, gated, err);
    switch (tile_tokens(M)) {
        case 16: return launch4<16, 4, 2>(a, codes, p, tiles_w, n_sms, stream);
        case 32: return launch4<32, 4, 2>(a, codes, p, tiles_w, n_sms, stream);
        case 64: return launch4<64, 4, 2>(a, codes, p, tiles_w, n_sms, stream);
        default: return launch4<128, 4, 1>(a, codes, p, tiles_w, n_sms, stream);
    }
}

// The same with the parameters in one array (the stream last): a call through ctypes costs 0.1 us a parameter.
TNX_EXPORT int tnx_gemm_mxfp4_16_packed(const long long* v) {
    return tnx_gemm_mxfp4_16((const void*)v[0], (long long)v[1], (const void*)v[2], (const void*)v[3], (const float*)v[4], (const float*)v[5],
                             (void*)v[6], (int)v[7], (long long)v[8], (int)v[9], (int)v[10], (int)v[11], (int)v[12], (int)v[13], (int)v[14],
                             (int*)v[15], (cudaStream_t)v[16]);
}
TNX_EXPORT int tnx_gemm_mxfp4_4_packed(const long long* v) {
    return tnx_gemm_mxfp4_4((const void*)v[0], (const void*)v[1], (const void*)v[2], (const void*)v[3], (const float*)v[4], (const float*)v[5],
                            (void*)v[6], (int)v[7], (long long)v[8], (int)v[9], (int)v[10], (int)v[11], (int)v[12], (int)v[13], (int)v[14],
                            (int*)v[15], (cudaStream_t)v[16]);
}
