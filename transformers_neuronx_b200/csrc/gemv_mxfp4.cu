// Products of a few tokens with a 4-bit matrix (formats: mxfp4.cuh; what is computed: gemm_mxfp4.cu).  The matrix is streamed once, straight
// into registers: no stage lies between memory and the multiplications.
//
// A warp takes 16 rows of W and walks K in chunks of 128 columns: four blocks of 32, one for each of the four lanes that share a row of
// an MMA (mma.sync m16n8k16).  Which column of K stands where in an MMA is free as long as both operands agree, so a lane multiplies
// its own block: 16 bytes of codes and one scale byte a row, loaded as they lie.  The block's eight magnitudes times its scale are a
// table in registers, bytes are looked up by permutation (15 instructions for eight values), and the lanes of a column find eight
// neighbouring activations of their block as one 16-byte piece in shared memory.
//
// Values and activations are multiplied as bfloat16, which holds a code times its scale exactly; activations of other types are the
// exact sum of two (float16) or three (32 bits) bfloat16 terms, which share the looked-up values.
//
// A block of eight warps: wf groups of 16 rows by 8 / wf shares of K, whose sums meet in shared memory; K may be split further over the
// blocks of a cluster.  More rows a block means activations are fetched less often, fewer that small matrices reach all SMs.
#include "mxfp4.cuh"

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int CHUNK = 128;                   // columns of K: four blocks
constexpr int AHEAD = 4;                     // chunks a warp has asked for

struct Params {
    const void* a; const uint8_t* a_scales; long long lda;
    int a_kind, a_vec;                       // 0: h16, 1: float, 2: codes; rows can be read 16 bytes at a time
    const uint8_t* codes; const uint8_t* scales;
    const float* bias; const float* residual; void* out; long long ldc;
    int M, N, K, w_rows, blocks, chunks, act, out_h16, gated;
    int wf, splits, chunks_per_split, phase; // phase: chunks whose activations lie in shared memory at a time
};

struct Table { uint32_t h0, h1, l0, l1; };
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    __nv_bfloat162 r = __hmul2(*(__nv_bfloat162*)&a, *(__nv_bfloat162*)&b);
    return *(uint32_t*)&r;
}
__device__ __forceinline__ Table make_table(uint32_t E) {
    uint32_t s = E ? E << 7 : 0x0040u;
    if (E == 255u) s = 0x7FC0u;
    s |= s << 16;
    const uint32_t p0 = mul_bf16x2(0x3F000000u, s), p1 = mul_bf16x2(0x3FC03F80u, s), p2 = mul_bf16x2(0x40404000u, s), p3 = mul_bf16x2(0x40C04080u, s);
    Table t;
    t.l0 = prmt(p0, p1, 0x6420); t.h0 = prmt(p0, p1, 0x7531);
    t.l1 = prmt(p2, p3, 0x6420); t.h1 = prmt(p2, p3, 0x7531);
    return t;
}
__device__ __forceinline__ void decode8(uint32_t w, const Table& t, uint32_t (&o)[4]) {
    const uint32_t s = w & 0x77777777u, s2 = s >> 16, w4 = w << 4;
    const uint32_t ha = prmt(t.h0, t.h1, s) | (prmt(w, w4, 0x9D8C) & 0x80808080u), la = prmt(t.l0, t.l1, s);
    const uint32_t hb = prmt(t.h0, t.h1, s2) | (prmt(w, w4, 0xBFAE) & 0x80808080u), lb = prmt(t.l0, t.l1, s2);
    o[0] = prmt(la, ha, 0x5140); o[1] = prmt(la, ha, 0x7362);
    o[2] = prmt(lb, hb, 0x5140); o[3] = prmt(lb, hb, 0x7362);
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *(uint32_t*)&r;
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Eight activations of a token from column k on as TERMS pieces of eight bfloat16 values whose sum they are; zeros behind the last column.
template <int TERMS>
__device__ __forceinline__ void load_terms(const Params& p, int token, int k, uint4 (&out)[TERMS]) {
    float v[8];
    if (p.a_kind == 2) {
        uint32_t c = 0u;
        float s = 0.f;
        if (k < p.blocks * 32) {
            const long long b = (long long)token * p.blocks + (k >> 5);
            c = *(const uint32_t*)((const uint8_t*)p.a + b * 16 + ((k & 31) >> 1));
            s = mx_scale(p.a_scales[b]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = mx_code(c >> (4 * j)) * s;
    } else if (p.a_kind == 0 && p.a_vec && k + 8 <= p.K) {
        const h16* src = (const h16*)p.a + token * p.lda + k;
        if (TERMS == 1) { out[0] = __ldg((const uint4*)src); return; }
        Vec8<h16> q;
        q.raw = __ldg((const uint4*)src);
        q.get(v);
    } else if (p.a_kind == 1 && p.a_vec && k + 8 <= p.K) {
        const float* src = (const float*)p.a + token * p.lda + k;
        const float4 x = __ldg((const float4*)src), y = __ldg((const float4*)src + 1);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = k + j >= p.K ? 0.f : p.a_kind ? ((const float*)p.a)[token * p.lda + k + j] : h16_to_float(((const h16*)p.a)[token * p.lda + k + j]);
    }
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
            const float2 r = unpack_bf16(w[j]);
            // what is not finite is whole in the first term (a rest would be NaN for an infinity)
            v[2 * j] = fabsf(r.x) < INFINITY ? v[2 * j] - r.x : 0.f;
            v[2 * j + 1] = fabsf(r.y) < INFINITY ? v[2 * j + 1] - r.y : 0.f;
        }
        out[t] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// NT: groups of eight tokens.
template <int TERMS, int NT>
__global__ void __launch_bounds__(THREADS, 2) gemv_kernel(const Params p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk_n = WARPS / p.wf, wf = warp % p.wf, wk = warp / p.wf;
    const int c_begin = (int)blockIdx.z * p.chunks_per_split, c_end = min(p.chunks, c_begin + p.chunks_per_split);
    // rows of W behind a lane's two MMA rows; gated: a gate row and its up row
    const int tile = blockIdx.x * p.wf + wf;
    const int ra = min(p.gated ? tile * 8 + g : tile * 16 + g, p.w_rows - 1);
    const int rb = min(p.gated ? p.N + tile * 8 + g : tile * 16 + 8 + g, p.w_rows - 1);
    const uint8_t* ca = p.codes + (long long)ra * p.blocks * 16 + t * 16;
    const uint8_t* cb = p.codes + (long long)rb * p.blocks * 16 + t * 16;
    const uint8_t* sa = p.scales + (long long)ra * p.blocks + t;
    const uint8_t* sb = p.scales + (long long)rb * p.blocks + t;

    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

    pdl_launch_dependents();
    pdl_wait();
    uint4* xs = (uint4*)smem;                             // [term][chunk of the phase][piece of a block][token][lane t]
    const int term_step = p.phase * 16 * p.M;
    for (int p0 = c_begin; p0 < c_end; p0 += p.phase) {
        const int p1 = min(c_end, p0 + p.phase);
        const int per = (p1 - p0 + wk_n - 1) / wk_n, b = min(p0 + wk * per, p1), e = min(b + per, p1);
        uint4 qa[AHEAD], qb[AHEAD];
        uint32_t ea[AHEAD], eb[AHEAD];
        auto load = [&](int j, int c) {
            const bool in = c < e && 4 * c + t < p.blocks;
            qa[j] = qb[j] = make_uint4(0u, 0u, 0u, 0u);
            ea[j] = eb[j] = 0u;
            if (in) {
                qa[j] = __ldg((const uint4*)(ca + (long long)c * 64));
                qb[j] = __ldg((const uint4*)(cb + (long long)c * 64));
                ea[j] = __ldg(sa + 4 * c);
                eb[j] = __ldg(sb + 4 * c);
            }
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) load(j, b + j);
        // this phase's activations: pieces of eight columns
        if (p0 != c_begin) __syncthreads();
        for (int i = threadIdx.x; i < (p1 - p0) * 16 * p.M; i += THREADS) {
            const int u = i % ((p1 - p0) * 16), token = i / ((p1 - p0) * 16);
            const int c = u >> 4, tt = (u >> 2) & 3, piece = u & 3;
            uint4 v[TERMS];
            load_terms<TERMS>(p, token, (p0 * 16 + u) * 8, v);
#pragma unroll
            for (int k = 0; k < TERMS; ++k) xs[k * term_step + ((c * 4 + piece) * p.M + token) * 4 + tt] = v[k];
        }
        __syncthreads();
        for (int c = b; c < e; c += AHEAD) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (c + j >= e) break;
                const Table ta = make_table(ea[j]), tb = make_table(eb[j]);
                const uint32_t wa[4] = {qa[j].x, qa[j].y, qa[j].z, qa[j].w}, wb[4] = {qb[j].x, qb[j].y, qb[j].z, qb[j].w};
                load(j, c + j + AHEAD);
                const uint4* xc = xs + (c + j - p0) * 16 * p.M;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t A[4], B[4];
                    decode8(wa[i], ta, A);
                    decode8(wb[i], tb, B);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const int token = n * 8 + g;
#pragma unroll
                        for (int k = 0; k < TERMS; ++k) {
                            uint4 x = make_uint4(0u, 0u, 0u, 0u);
                            if (token < p.M) x = xc[k * term_step + (i * p.M + token) * 4 + t];
                            mma(acc[n], A[0], B[0], A[1], B[1], x.x, x.y);
                            mma(acc[n], A[2], B[2], A[3], B[3], x.z, x.w);
                        }
                    }
                }
            }
        }
    }
    // The shares' sums: [share][token][rows + 4], the lanes of a warp in 32 banks.
    const int rows = p.wf * 16, ld = rows + 4;
    float* red = (float*)smem;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int token = n * 8 + 2 * t + (j & 1);
            if (token < p.M) red[(wk * p.M + token) * ld + wf * 16 + g + 8 * (j >> 1)] = acc[n][j];
        }
    const int splits = p.splits, rank = splits > 1 ? (int)cta_rank() : 0;
    if (splits > 1) cluster_sync(); else __syncthreads();
    auto total = [&](int token, int row) {                // shares in their order, then the cluster's blocks in theirs
        float v = 0.f;
        for (int s = 0; s < splits; ++s)
            for (int w = 0; w < wk_n; ++w) {
                const float* at = red + (w * p.M + token) * ld + row;
                v += splits > 1 ? ld_cluster(at, (uint32_t)s) : *at;
            }
        return v;
    };
    const int feats = p.gated ? rows / 2 : rows;
    for (int i = threadIdx.x * splits + rank; i < feats * p.M; i += THREADS * splits) {
        const int f = i % feats, token = i / feats, n = blockIdx.x * feats + f;
        if (n >= p.N) continue;
        const long long o = (long long)token * p.ldc + n;
        const float res = p.residual ? __ldcg(p.residual + o) : 0.f;
        float v;
        if (p.gated) {
            const int row = (f >> 3) * 16 + (f & 7);
            float gate = total(token, row), up = total(token, row + 8);
            if (p.bias) { gate += __ldg(p.bias + n); up += __ldg(p.bias + p.N + n); }
            v = apply_activation(gate, p.act) * up;
        } else {
            v = total(token, f);
            if (p.bias) v += __ldg(p.bias + n);
            v = apply_activation(v, p.act);
        }
        v += res;
        if (p.out_h16) ((h16*)p.out)[o] = float_to_h16(v);
        else ((float*)p.out)[o] = v;
    }
    if (splits > 1) cluster_sync();                       // no block leaves while its sums may still be read
}

constexpr int SMEM_MOST = 96 * 1024;

template <int TERMS, int NT>
int launch(const Params& p, int smem, cudaStream_t stream) {
    static TnxSmemLimit limit;
    auto kernel = gemv_kernel<TERMS, NT>;
    const int r = limit.allow(kernel, SMEM_MOST);
    if (r) return r;
    const int per = (p.gated ? 8 : 16) * p.wf;
    const dim3 grid((p.N + per - 1) / per, 1, p.splits);
    if (p.splits > 1) return tnx_launch_cluster(1, dim3(1, 1, p.splits), kernel, grid, dim3(THREADS), smem, stream, p);
    return tnx_launch_ex(1, kernel, grid, dim3(THREADS), smem, stream, p);
}
template <int TERMS>
int launch_terms(const Params& p, int smem, cudaStream_t stream) {
    if (p.M <= 8) return launch<TERMS, 1>(p, smem, stream);
    if (p.M <= 16) return launch<TERMS, 2>(p, smem, stream);
    return launch<TERMS, 4>(p, smem, stream);
}

int g_forced_wf = 0, g_forced_splits = 0;

}  // namespace

constexpr int FEW_TOKENS = 32;
TNX_EXPORT int tnx_gemv_mxfp4_tokens() { return FEW_TOKENS; }
// For sweeps and tests: groups of 16 rows a block (1, 2, 4 or 8) and the split of K (1, 2, 4 or 8) whatever the sizes (0: the plan's own).
TNX_EXPORT void tnx_gemv_mxfp4_force(int wf, int splits) { g_forced_wf = wf; g_forced_splits = splits; }

// a_kind: 0 16-bit, 1 32-bit activations (pitch lda), 2 codes (4-byte aligned) with a_scales; codes of W 16-byte aligned.
TNX_EXPORT int tnx_gemv_mxfp4(const void* a, int a_kind, const void* a_scales, long long lda, const void* codes, const void* scales, const float* bias,
                              const float* residual, void* out, int out_h16, long long ldc, int M, int N, int K, int act, int gated, int n_sms,
                              cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || a_kind < 0 || a_kind > 2 || act < 0 || act >= TNX_ACT_COUNT || n_sms <= 0) return TNX_ERR_BAD_ARG;
    if (M > FEW_TOKENS || ((uintptr_t)codes & 15) || (a_kind == 2 && ((uintptr_t)a & 3))) return TNX_ERR_UNSUPPORTED;
    Params p;
    p.a = a; p.a_scales = (const uint8_t*)a_scales; p.lda = lda; p.a_kind = a_kind;
    p.a_vec = ((uintptr_t)a & 15) == 0 && lda % (a_kind == 1 ? 4 : 8) == 0;
    p.codes = (const uint8_t*)codes; p.scales = (const uint8_t*)scales; p.bias = bias; p.residual = residual; p.out = out; p.ldc = ldc;
    p.M = M; p.N = N; p.K = K; p.w_rows = gated ? 2 * N : N; p.blocks = (K + MX_BLOCK - 1) / MX_BLOCK; p.chunks = (p.blocks + 3) / 4;
    p.act = act; p.out_h16 = out_h16; p.gated = gated;
#ifdef TNX_F16
    const int terms = a_kind == 2 ? 1 : a_kind == 1 ? 3 : 2;
#else
    const int terms = a_kind == 1 ? 3 : 1;
#endif
    p.wf = g_forced_wf ? g_forced_wf : M <= 2 ? 1 : M <= 4 ? 2 : M <= 8 ? 4 : 8;
    const int per = (gated ? 8 : 16) * p.wf;
    const long long tiles = (N + per - 1) / per;
    p.splits = 1;
    while (p.splits < 8 && tiles * p.splits < 2 * n_sms && p.chunks >= 2 * p.splits * (WARPS / p.wf)) p.splits *= 2;
    if (g_forced_splits) p.splits = g_forced_splits;
    p.chunks_per_split = (p.chunks + p.splits - 1) / p.splits;
    while (p.splits > 1 && p.chunks_per_split * (p.splits - 1) >= p.chunks) { p.splits /= 2; p.chunks_per_split = (p.chunks + p.splits - 1) / p.splits; }
    // a phase's activations: 256 bytes a chunk, token and term
    const int chunk_bytes = CHUNK * 2 * M * terms, most = SMEM_MOST / chunk_bytes;
    const int phases = (p.chunks_per_split + most - 1) / most;
    p.phase = (p.chunks_per_split + phases - 1) / phases;
    const int x_bytes = p.phase * chunk_bytes, red = WARPS / p.wf * M * (p.wf * 16 + 4) * 4;
    const int smem = x_bytes > red ? x_bytes : red;
    if (terms == 1) return launch_terms<1>(p, smem, stream);
    if (terms == 2) return launch_terms<2>(p, smem, stream);
    return launch_terms<3>(p, smem, stream);
}
