// Projection with both operands in microscaled 4-bit floating point (formats: fp4.cuh), on the block-scaled tensor cores:
//
//   y[m, n] = epilogue( gx[m] * gw[n] * sum_k q_x[m, k] s_x[m, k / block] q_w[n, k] s_w[n, k / block] )
//
// A stage of either kernel's ring holds 256 elements of K (128 bytes a row) of both operands, by TMA in the 128-byte swizzle that the
// MMA reads, and their scale tiles, which lie in memory as tensor memory wants them.  The MMA thread copies a stage's
// scales to tensor memory and issues its MMAs of 64 k behind them; both run in issue order, and a stage's columns of
// scales are written again only when its MMAs are known to be done (the stage's `empty` barrier).
//
// Few tokens (stream kernel): the weight is operand A (128 output channels: the lanes of the accumulator), the tokens are
// operand B (the columns), so that one token costs a tile of 128 x 16 and not one of 128 x 128; K is split over the CTAs of a cluster
// where the channels alone do not fill the GPU.  Many tokens (pair kernel): tokens are operand A, CTA pairs on tiles of
// 256 x 256 or 256 x 128, persistent.  All waits are bounded (umma.cuh).
#include <cooperative_groups.h>

#include "fp4_encode.cuh"
#include "umma.cuh"

namespace cg = cooperative_groups;

namespace rwkv7 {
namespace f4 {
constexpr int KS = 256, KSB = 128;  // elements and bytes of K a stage
constexpr int tiles_per_stage(int format) { return format == fp4::MX ? 2 : 4; }  // scale tiles of 128 rows
constexpr int sf_bytes(int format) { return tiles_per_stage(format) * fp4::SCALE_TILE_BYTES; }
constexpr int BAR_BYTES = 1024;
constexpr int pow2_cols(int need) {
    int c = 32;
    while (c < need) c *= 2;
    return c;
}
}  // namespace f4

struct Fp4Args {
    const float *wg, *xg;  // row factors (nvfp4; NULL = 1)
    const void *bias, *residual;
    const void* x;  // FUSED: the tokens, not quantised yet, ldx elements apart
    int64_t ldx;
    void* y;
    int M, N, K;
    int relu2;
    int vec;     // rows of y and the residual allow 16-byte accesses
    int splits;  // stream kernel: CTAs of a cluster that share a K range
    int tiles_m, tiles_n;
    unsigned int* error;
};
struct Fp4Maps {
    CUtensorMap w, x, ws, xs, y;  // codes, scale tiles, and (pair kernel) the output
};

// Instruction descriptor of the block-scaled 4-bit kinds: E2M1 operands (1), scale type (0 = E4M3, 1 = E8M0), and which
// byte of a scale word the first block of this K step has (0, or 2 for the second half of a word with two scales a step).
__host__ __device__ constexpr uint32_t fp4_idesc(int M, int N, int e8m0, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)e8m0 << 23) | ((uint32_t)(M >> 7) << 27) | (sf_id << 29);
}
template <int FORMAT, int GROUP>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define RWKV7_FP4_MMA(KIND)                                                                              \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                        \
                 "tcgen05.mma.cta_group::%7." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"               \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "n"(GROUP) : "memory")
    if constexpr (FORMAT == fp4::MX) RWKV7_FP4_MMA("kind::mxf4.block_scale.scale_vec::2X");
    else RWKV7_FP4_MMA("kind::mxf4nvf4.block_scale.scale_vec::4X");
#undef RWKV7_FP4_MMA
}
// Descriptor of a scale tile (32 rows of 16 bytes, 8-row groups 128 bytes apart, no swizzle), and its copy to four columns,
// repeated in the four lane quarters
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
template <int GROUP> __device__ __forceinline__ void copy_scale_tile(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::%2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc), "n"(GROUP) : "memory");
}
// relu(y)^2, NaN stays
__device__ __forceinline__ float relu_squared(float y) {
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(y));
    return r * r;
}
__device__ __forceinline__ bool elect_lane() {  // (the compiler knows that one thread runs what this guards)
    uint32_t pred;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.b32 %0, 1, 0, P;\n\t}" : "=r"(pred));
    return pred != 0;
}

// The scale copies and MMAs of one stage, `steps` of 64 k of it (4, fewer at a ragged end).  BR: scale tiles of operand B beside one another.
template <int FORMAT, int GROUP, int M, int N, int BR>
__device__ __forceinline__ void issue_stage(uint32_t d, uint64_t da, uint64_t db, uint32_t sfa, uint64_t sf_a, uint64_t sf_b, int steps, bool first) {
    constexpr int TPS = f4::tiles_per_stage(FORMAT);
    constexpr uint32_t id0 = fp4_idesc(M, N, FORMAT == fp4::MX, 0), id2 = fp4_idesc(M, N, 1, 2);
    const uint32_t sfb = sfa + TPS * 4;
#pragma unroll
    for (int t = 0; t < TPS; ++t) {
        copy_scale_tile<GROUP>(sfa + 4 * t, sf_a + (uint64_t)(t * (fp4::SCALE_TILE_BYTES >> 4)));
#pragma unroll
        for (int r = 0; r < BR; ++r)
            copy_scale_tile<GROUP>(sfb + 4 * (t * BR + r), sf_b + (uint64_t)((r * TPS + t) * (fp4::SCALE_TILE_BYTES >> 4)));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int t = FORMAT == fp4::MX ? j >> 1 : j;
        if (j < steps)
            umma_fp4<FORMAT, GROUP>(d, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), FORMAT == fp4::MX && (j & 1) ? id2 : id0, sfa + 4 * t,
                                    sfb + 4 * BR * t, first && j == 0 ? 0u : 1u);
    }
}

// ---------------------------------------------------------------- few tokens
namespace fs {
constexpr int BM = 128, EW = 8, THREADS = 64 + 32 * EW, A_BYTES = BM * f4::KSB, MAX_SPLITS = 4;  // (four tokens a CTA at least)
constexpr int tokens_at_once(int bn) { return bn >= 64 ? 16 : 8; }  // of an epilogue warp
constexpr int FUSED_STAGES = 16;  // of tokens, which stay, where the kernel quantises them itself
constexpr int ring_bytes(int format) { return A_BYTES + f4::sf_bytes(format); }                    // a stage of the weight
constexpr int token_bytes(int format, int bn) { return bn * f4::KSB + f4::sf_bytes(format); }      // and one of tokens
// DEEP: as many stages as fit, for grids of at most a CTA an SM; else room for two CTAs an SM where the tile is narrow
constexpr int stages(int bn, bool deep) { return bn == 16 ? (deep ? 8 : 4) : bn == 32 ? (deep ? 8 : 3) : bn == 64 ? 6 : 4; }
constexpr int q_bytes(int bn) { return BM * 4 * (bn + 4 * MAX_SPLITS); }  // partial sums of a tile
constexpr int smem_bytes(int format, int bn, bool deep, bool fused) {
    return stages(bn, deep) * ring_bytes(format) + (fused ? FUSED_STAGES : stages(bn, deep)) * token_bytes(format, bn) + q_bytes(bn) + f4::BAR_BYTES +
           bn * 4 + 1024;
}
constexpr int sf_cols(int format) { return f4::tiles_per_stage(format) * 8; }
constexpr int tmem_cols(int format, int bn, bool deep) { return f4::pow2_cols(bn + stages(bn, deep) * sf_cols(format)); }
}  // namespace fs

// FUSED: the epilogue's threads make the tokens' operand themselves, codes in the 128-byte swizzle and scale tiles as the quantiser would
// write them, for the K range of this CTA (stages kb0 .. kb0 + nk; nvfp4 needs the largest magnitude of whole rows for it).  `team` threads a row, 32 at
// least; what lies beyond K is zero.  red: 8 floats.
template <int FORMAT, typename T>
__device__ __forceinline__ void quantise_tokens(const T* x, int64_t ldx, int M, int K, int kb0, int nk, unsigned char* codes, unsigned char* scales,
                                                float* factor, float* red) {
    constexpr int SF = f4::sf_bytes(FORMAT), THREADS = 32 * fs::EW, BN = 16;
    const int tid = threadIdx.x - 64, lane = tid & 31;
    int team = THREADS;
    while (team > 32 && THREADS / team < M) team /= 2;
    const int at = tid % team, pieces = K / 16;
    for (int r0 = 0; r0 < M; r0 += THREADS / team) {
        const int row = r0 + tid / team;
        const bool live = row < M;
        const T* xr = x + (live ? row : 0) * ldx;
        int ge = 127;
        if constexpr (FORMAT == fp4::NV) {
            float m = 0.0f;
#pragma unroll 4
            for (int p = at; p < pieces; p += team) {
                const Piece<T> one = load_piece<T>(xr + 16 * p);
                m = fmaxf(m, finite_amax(one, piece_amax(one)));
            }
            m = group_max<32>(m);
            if (team > 32) {
                asm volatile("bar.sync 1, 256;" ::: "memory");  // (the last rows' maxima have been read)
                if (lane == 0) red[tid >> 5] = m;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                for (int w = tid / team * (team / 32), n = team / 32; n > 0; ++w, --n) m = fmaxf(m, red[w]);
            }
            const int e = max(__float_as_int(m) >> 23, 1);
            ge = m > 0.0f ? max(e - 10, 1) : 127;
            if (at == 0 && live) factor[row] = __int_as_float(ge << 23);
        } else if (at == 0 && live) {
            factor[row] = 1.0f;
        }
#pragma unroll 2
        for (int i0 = at - lane; i0 < 16 * nk; i0 += team) {  // (whole warps)
            const int i = i0 + lane, p = 16 * kb0 + i;
            Piece<T> piece{};
            if (p < pieces) piece = load_piece<T>(xr + 16 * p);
            uint2 c;
            const uint32_t byte = encode_piece<T, FORMAT>(piece, piece_amax(piece), ge, c);
            if (live && i < 16 * nk) {
                const int stage = i >> 4, j = i & 15;  // a piece: 8 bytes of the row's 128
                *reinterpret_cast<uint2*>(codes + stage * (BN * f4::KSB) + row * f4::KSB + (((j >> 1) ^ (row & 7)) << 4) + (j & 1) * 8) = c;
                const int block = FORMAT == fp4::NV ? j : j >> 1;
                if (FORMAT == fp4::NV || !(j & 1))
                    scales[stage * SF + (block >> 2) * fp4::SCALE_TILE_BYTES + row * 16 + (block & 3)] = (unsigned char)(p < pieces ? byte : 0);
            }
        }
    }
    fence_proxy_async_smem();
}

// grid (channel tiles, token tiles, splits); warp 0 = producer, warp 1 = MMA, warps 2..9 = epilogue (two a lane quarter,
// in turn).  A lane is a channel: what a warp stores or reads for one token is 32 neighbouring channels, whole sectors.
// The kernel before this one in the stream is the quantiser of the tokens: only their codes, scales and row factors wait for
// it.  It has itself waited for everything earlier before it let this kernel start, so the weight, bias and residual are there.
// FUSED: there is no quantiser, the tokens are quantised here under the first loads of the weight (quantise_tokens); everything waits for the
// kernel before.
// Bound by the weight's way from memory where there is much of it, else by the launch, the quantiser and the chain load, MMA, exchange, store.  us a
// call, weights out of memory, nvfp4: 1 x 4096 -> 65536 (151 MB) 27.6 = 5.5 TB/s, 1 x 4096 -> 16384 (37.7 MB) 9.8, 1 x 4096 -> 4096
// 5.7, 64 x 4096 -> 4096 8.3, 64 x 4096 -> 16384 12.6, 64 x 16384 -> 4096 14.7.
template <int FORMAT, typename T, int BN, bool DEEP, bool FUSED>
__global__ void __launch_bounds__(fs::THREADS, DEEP ? 1 : 2) fp4_stream_kernel(const __grid_constant__ Fp4Maps maps, const Fp4Args p) {
    using namespace fs;
    constexpr int STAGES = stages(BN, DEEP), SF = f4::sf_bytes(FORMAT), TMEM_COLS = tmem_cols(FORMAT, BN, DEEP);
    constexpr int TOKEN_STAGES = FUSED ? FUSED_STAGES : STAGES, STAGE_BYTES = ring_bytes(FORMAT) + (FUSED ? 0 : token_bytes(FORMAT, BN));
    constexpr int TB = tokens_at_once(BN);
    static_assert(BN + STAGES * sf_cols(FORMAT) <= TMEM_COLS && TMEM_COLS <= 512, "tensor memory");
    static_assert(smem_bytes(FORMAT, BN, DEEP, FUSED) <= (DEEP ? 227 : 113) * 1024, "shared memory");
    static_assert(DEEP || TMEM_COLS <= 256, "tensor memory for two");
    extern __shared__ unsigned char smem_unaligned[];
    unsigned char* sm = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    // [A of all stages][B of all stages][scales of A][scales of B][partial sums: split, channel, token][barriers][row factors]
    unsigned char* sm_b = sm + STAGES * A_BYTES;
    unsigned char* sm_s = sm_b + TOKEN_STAGES * BN * f4::KSB;
    unsigned char* sm_t = sm_s + STAGES * SF;
    float* Q = reinterpret_cast<float*>(sm_t + TOKEN_STAGES * SF);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm_t + TOKEN_STAGES * SF + q_bytes(BN));
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* tokens_full = acc_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tokens_full + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* s_xg = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(full) + f4::BAR_BYTES);
    const AbortCtx actx{abort_flag, p.error};

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = tid & 31;
    const int n0 = blockIdx.x * BM, m0 = blockIdx.y * BN;
    const int all = (p.K + f4::KS - 1) / f4::KS, split = blockIdx.z;
    const int kb0 = split * all / p.splits, nk = (split + 1) * all / p.splits - kb0;  // at least one stage each
    const bool clustered = p.splits > 1;

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        mbar_init(acc_full, 1);
        mbar_init(tokens_full, 1);
        *abort_flag = 0;
        mbar_fence_init();
        if constexpr (FUSED) {
            tma_prefetch_desc(&maps.w), tma_prefetch_desc(&maps.ws);
        } else {
            // the weight does not depend on the kernel before this one: what the ring holds is requested under it
            for (int i = 0; i < STAGES && i < nk; ++i) {
                mbar_expect_tx(&full[i], STAGE_BYTES);
                tma_load_2d(sm + i * A_BYTES, &maps.w, &full[i], (kb0 + i) * f4::KSB, n0);
                tma_load_2d(sm_s + i * SF, &maps.ws, &full[i], (kb0 + i) * (SF / 8), blockIdx.x);
            }
            tma_prefetch_desc(&maps.x), tma_prefetch_desc(&maps.xs);
        }
    }
    if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    cg::cluster_group cl = cg::this_cluster();
    if (clustered) cluster_arrive_relaxed();  // this CTA runs: the others may write into its partial sums

    // this thread's channel in the epilogue, its factor and bias
    const int q = warp & 3, half = (warp - 2) >> 2, ch = q * 32 + lane, n = n0 + ch;
    const int rows = min(BN, p.M - m0);
    float gw = 1.0f, bias = 0.0f;
    const int per = BN / p.splits, lg_per = 31 - __clz(per), pitch = per + 4;  // tokens that a CTA finishes; four more: no two lanes' 16 bytes meet in a bank

    if (warp == 0) {
        if (elect_lane()) {
            grid_dependency_wait();
            grid_launch_dependents();
            for (int i = 0; i < nk; ++i) {
                const int s = i % STAGES, kb = kb0 + i;
                if (i >= STAGES && !mbar_wait(&empty[s], ((i / STAGES) - 1) & 1, actx, kErrWaitEmpty)) break;
                if (FUSED || i >= STAGES) {
                    mbar_expect_tx(&full[s], STAGE_BYTES);
                    tma_load_2d(sm + s * A_BYTES, &maps.w, &full[s], kb * f4::KSB, n0);
                    tma_load_2d(sm_s + s * SF, &maps.ws, &full[s], kb * (SF / 8), blockIdx.x);
                }
                if constexpr (!FUSED) {
                    tma_load_2d(sm_b + s * BN * f4::KSB, &maps.x, &full[s], kb * f4::KSB, m0);
                    tma_load_2d(sm_t + s * SF, &maps.xs, &full[s], kb * (SF / 8), m0 / 128);
                }
            }
        }
    } else if (warp == 1) {
        if (elect_lane()) {
            bool ok = !FUSED || mbar_wait_hot(tokens_full, 0, actx, kErrWaitFull);
            for (int i = 0; ok && i < nk; ++i) {
                const int s = i % STAGES, t = FUSED ? i : s;
                if (!mbar_wait_hot(&full[s], (i / STAGES) & 1, actx, kErrWaitFull)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                issue_stage<FORMAT, 1, BM, BN, 1>(tmem, make_sw128_kmajor_desc(smem_u32(sm + s * A_BYTES)),
                                                  make_sw128_kmajor_desc(smem_u32(sm_b + t * BN * f4::KSB)), tmem + BN + s * sf_cols(FORMAT),
                                                  scale_desc(smem_u32(sm_s + s * SF)), scale_desc(smem_u32(sm_t + t * SF)),
                                                  (p.K - (kb0 + i) * f4::KS + 63) / 64, i == 0);
                tc_commit(&empty[s]);
            }
            if (ok) tc_commit(acc_full);
        }
    } else {
        if constexpr (FUSED) {
            grid_dependency_wait();
            quantise_tokens<FORMAT, T>(static_cast<const T*>(p.x), p.ldx, rows, p.K, kb0, nk, sm_b, sm_t, s_xg,
                                       reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(full) + f4::BAR_BYTES / 2));
        }
        if (n < p.N) {
            if (p.wg) gw = p.wg[n];
            if (p.bias) bias = to_f<T>(static_cast<const T*>(p.bias)[n]);
        }
        if constexpr (!FUSED) {
            grid_dependency_wait();
            for (int t = tid - 64; t < rows; t += 32 * EW) s_xg[t] = p.xg ? p.xg[m0 + t] : 1.0f;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (FUSED && tid == 64) mbar_arrive(tokens_full);
        bool ok = true;
        if (lane == 0) ok = mbar_wait(acc_full, 0, actx, kErrWaitDFull);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (clustered) cluster_wait();
        if (ok) {
            tc_fence_after();
            const T* res = p.residual ? static_cast<const T*>(p.residual) + (size_t)m0 * p.N + min(n, p.N - 1) : nullptr;
            T* out = static_cast<T*>(p.y) + (size_t)m0 * p.N + n;
#pragma unroll 1
            for (int c = TB * half; c < rows; c += 2 * TB) {
                // (residual reads are clamped to tokens and channels that exist, so that they need no branch and stay in flight together)
                T r[TB];
#pragma unroll
                for (int i = 0; i < TB; ++i) r[i] = from_f<T>(0.0f);
                if (res && !clustered) {
#pragma unroll
                    for (int i = 0; i < TB; ++i) r[i] = res[(size_t)min(c + i, rows - 1) * p.N];
                }
                uint32_t v[TB];
                if constexpr (TB == 16) tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
                else tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + c, v);
                tc_wait_ld();
                if (!clustered) {
#pragma unroll
                    for (int i = 0; i < TB; ++i) {
                        float y = fmaf(__uint_as_float(v[i]), gw * s_xg[c + i], bias);
                        if (p.relu2) y = relu_squared(y);
                        if (c + i < rows && n < p.N) out[(size_t)(c + i) * p.N] = from_f<T>(y + to_f<T>(r[i]));
                    }
                } else {
                    // four tokens at a time to the CTA that finishes them (64 tokens, four CTAs: 24 KB leave a CTA at 14 bytes a cycle, which is what bounds
                    // this; single words took a quarter longer)
#pragma unroll
                    for (int i = 0; i < TB; i += 4) {
                        const int to = (c + i) >> lg_per;
                        if (c + i < rows)
                            *reinterpret_cast<uint4*>(cl.map_shared_rank(Q, to) + (split * BM + ch) * pitch + (c + i) - (to << lg_per)) =
                                make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                }
            }
            tc_fence_before();
        }
    }
    __syncwarp();
    if (clustered) {
        if (warp < 2) cluster_wait();
        // four tokens of this thread's channel a turn (one body: code that runs once waits for its instructions): the partial sums in the order of K, the
        // residual two turns ahead
        const int t0 = split << lg_per, count = min(rows - t0, per);
        const T* res = p.residual ? static_cast<const T*>(p.residual) + (size_t)(m0 + t0) * p.N + min(n, p.N - 1) : nullptr;
        T r[3][4];
        const auto request = [&](T (&to)[4], int t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                to[i] = from_f<T>(0.0f);
                if (res && t < count) to[i] = res[(size_t)min(t + i, count - 1) * p.N];  // (clamped to what exists: all four stay in flight)
            }
        };
        if (warp >= 2) request(r[0], 4 * half), request(r[1], 4 * half + 8);
        cl.sync();
        if (warp >= 2 && n < p.N && *abort_flag == 0) {  // (the producer and MMA warps, and channels beyond N, have no token)
#pragma unroll 1
            for (int t = 4 * half; t < count; t += 8) {
                request(r[2], t + 16);
                const float* src = Q + ch * pitch + t;
                float4 sum = *reinterpret_cast<const float4*>(src);
                for (int z = 1; z < p.splits; ++z) {
                    const float4 more = *reinterpret_cast<const float4*>(src + z * BM * pitch);
                    sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
                }
                const float4 gx = *reinterpret_cast<const float4*>(s_xg + t0 + t);
                const float a[4] = {sum.x, sum.y, sum.z, sum.w}, g[4] = {gx.x, gx.y, gx.z, gx.w};
                T* out = static_cast<T*>(p.y) + (size_t)(m0 + t0 + t) * p.N + n;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float y = fmaf(a[i], gw * g[i], bias);
                    if (p.relu2) y = relu_squared(y);
                    if (t + i < count) *out = from_f<T>(y + to_f<T>(r[0][i]));
                    out += p.N;
                    r[0][i] = r[1][i], r[1][i] = r[2][i];
                }
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// ---------------------------------------------------------------- many tokens
// Roles and barriers as in gemm_umma_pair_kernel (gemm_umma.cu): both producers' loads complete on the leader's full[s]; the
// leader's commits arrive on empty[s] / acc_full[a] in both CTAs; the epilogue warps of both arrive on the leader's acc_empty[a].
// Each CTA stages its own 128 token rows, half of the channels, the scales of its own rows and those of all channels
// (each CTA's tensor memory needs them).  Eight epilogue warps, two a lane quarter, each with half of the columns.
// A pair reads 64 KB a stage of 256 k for 512 cycles of MMA: bound by the way from L2 into shared memory (54 to 75 bytes a cycle and SM) and, in
// long products, by the power cap.  Device us, quantiser included, fp16 out: 8192 x 4096 -> 16384 nvfp4 243 to 267 (1.1 TFLOP; the quantiser 20 of it: 4.9
// PFLOP/s, three times the measured bf16 rate), mxfp4 232; 2048 x 4096 -> 16384 65.8; 777 x 2560 -> 10240 22.6 and 20.2 (160 tiles on 74 pairs: three
// turns, the last one for 12).
namespace fp {
constexpr int BM = 128, PAIR_M = 256, EW = 8, THREADS = 64 + 32 * EW, STAGES = 5, A_BYTES = BM * f4::KSB, GROUP_M = 16;
constexpr int b_bytes(int bn) { return bn / 2 * f4::KSB; }
constexpr int sfb_rows(int bn) { return bn / 128; }
constexpr int stage_bytes(int format, int bn) { return A_BYTES + b_bytes(bn) + (1 + sfb_rows(bn)) * f4::sf_bytes(format); }
constexpr int accs(int bn) { return bn == 256 ? 1 : 2; }
constexpr int sf_cols(int format, int bn) { return f4::tiles_per_stage(format) * 4 * (1 + sfb_rows(bn)); }
constexpr int STG_WARP_BYTES = 4096;  // 32 rows x 128 bytes
constexpr int vec_bytes(int bn) { return 2 * bn * 4; }  // channel factors and bias of a tile
constexpr int smem_bytes(int format, int bn) { return STAGES * stage_bytes(format, bn) + EW * STG_WARP_BYTES + f4::BAR_BYTES + vec_bytes(bn) + 1024; }
constexpr int TMEM_COLS = 512;
}  // namespace fp

__device__ __forceinline__ void fp4_tile(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int per_band = fp::GROUP_M * tiles_n, band = tile / per_band, within = tile - band * per_band;
    const int rows = min(fp::GROUP_M, tiles_m - band * fp::GROUP_M);
    tn = within / rows;
    tm = band * fp::GROUP_M + (within - tn * rows);
}

// The residual of 64 columns of a warp's 32 rows on its way into the warp's staging tile (16-bit types, aligned rows), eight lanes a
// row, whole lines; zeros where there is none.  The last copy out of the tile is awaited before.
__device__ __forceinline__ void request_residual(const Fp4Args& p, int row0, int col0, int lane, unsigned char* stg) {
    if (row0 >= p.M || col0 >= p.N) return;  // (nobody would wait for it before the next request)
    if (lane == 0) tma_store_wait_read<0>();
    __syncwarp();
    const int col = col0 + (lane & 7) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = (lane >> 3) + 4 * i, row = row0 + r;
        const bool here = row < p.M && col < p.N;
        const uint16_t* src = static_cast<const uint16_t*>(p.residual) + (here ? (size_t)row * p.N + col : 0);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     ::"r"(smem_u32(stg + r * 128 + (((lane & 7) ^ (r & 7)) << 4))), "l"(src), "r"(here ? 16 : 0) : "memory");
    }
}

// 64 columns of a warp's 32 rows (a lane is a row): factors and bias, then MODE 0 nothing, 1 relu^2, 2 + residual.  16-bit
// results go through the warp's staging tile (16-byte pieces xored by the row: the layout of a 128-byte-swizzled tensor map) and
// leave as one bulk copy, or, where rows of y are not 16-byte aligned, as coalesced single values.  The residual
// comes in by the same tile (request_residual): a lane that reads its own row from memory touches 32 lines an instruction.
template <int FORMAT, typename T, int MODE>
__device__ __forceinline__ void fp4_columns(const Fp4Args& p, const CUtensorMap& tm_y, const uint32_t (&v)[64], const float* wg, const float* bias, float gx,
                                            int row0, int col0, int lane, unsigned char* stg) {
    const int row = row0 + lane, live = row < p.M ? p.N - col0 : 0;  // columns of this row that exist
    const size_t o = (size_t)row * p.N + col0;
    const T* res = static_cast<const T*>(p.residual) + o;
    if (sizeof(T) == 2) {
        if (MODE == 2 && p.vec) asm volatile("cp.async.wait_all;" ::: "memory");
        else if (p.vec && lane == 0) tma_store_wait_read<0>();  // the last group's copy has left the staging tile
        __syncwarp();
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        float f[8], r[8];
        if constexpr (MODE == 2) {
            if (sizeof(T) == 2 && p.vec) {
                load8<T>(reinterpret_cast<const T*>(stg + lane * 128 + ((u ^ (lane & 7)) << 4)), r);
            } else if (p.vec) {
                if (8 * u < live) load8<T>(res + 8 * u, r);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = 8 * u + e < live ? to_f<T>(res[8 * u + e]) : 0.0f;
            }
        }
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias + 8 * u + h);
            f[h] = b.x, f[h + 1] = b.y, f[h + 2] = b.z, f[h + 3] = b.w;
            if constexpr (FORMAT == fp4::NV) {
                const float4 w = *reinterpret_cast<const float4*>(wg + 8 * u + h);
                f[h] = fmaf(__uint_as_float(v[8 * u + h]), gx * w.x, f[h]), f[h + 1] = fmaf(__uint_as_float(v[8 * u + h + 1]), gx * w.y, f[h + 1]);
                f[h + 2] = fmaf(__uint_as_float(v[8 * u + h + 2]), gx * w.z, f[h + 2]), f[h + 3] = fmaf(__uint_as_float(v[8 * u + h + 3]), gx * w.w, f[h + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[h + e] += __uint_as_float(v[8 * u + h + e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (MODE == 1) f[e] = relu_squared(f[e]);
            if constexpr (MODE == 2) f[e] += r[e];
        }
        if constexpr (sizeof(T) == 2) {
            store8<T>(reinterpret_cast<T*>(stg + lane * 128 + ((u ^ (lane & 7)) << 4)), f);
        } else {
            T* y = static_cast<T*>(p.y) + o + 8 * u;
            if (p.vec) {
                if (8 * u < live) store8<T>(y, f);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (8 * u + e < live) y[e] = from_f<T>(f[e]);
            }
        }
    }
    if constexpr (sizeof(T) == 2) {
        if (p.vec) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(&tm_y, stg, col0, row0);
                tma_store_commit();
            }
        } else {
            __syncwarp();
            const int cols = p.N - col0 < 64 ? p.N - col0 : 64, rows = p.M - row0 < 32 ? p.M - row0 : 32;
            for (int r = 0; r < rows; ++r)
                for (int c = lane; c < cols; c += 32)
                    static_cast<T*>(p.y)[(size_t)(row0 + r) * p.N + col0 + c] = *reinterpret_cast<const T*>(stg + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
            __syncwarp();
        }
    }
}

template <int FORMAT, typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(fp::THREADS, 1) fp4_pair_kernel(const __grid_constant__ Fp4Maps maps, const Fp4Args p) {
    using namespace fp;
    constexpr int SF = f4::sf_bytes(FORMAT), SFR = sfb_rows(BN), STAGE_BYTES = stage_bytes(FORMAT, BN), ACCS = accs(BN), B_BYTES = b_bytes(BN);
    static_assert(ACCS * BN + STAGES * sf_cols(FORMAT, BN) <= TMEM_COLS, "tensor memory");
    static_assert(smem_bytes(FORMAT, BN) <= 227 * 1024, "shared memory");
    extern __shared__ unsigned char smem_unaligned[];
    unsigned char* sm = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    // [A of all stages][B of all stages][output staging][scales of all stages][barriers][channel factors, bias]
    unsigned char* sm_b = sm + STAGES * A_BYTES;
    unsigned char* sm_o = sm_b + STAGES * B_BYTES;
    unsigned char* sm_s = sm_o + EW * STG_WARP_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm_s + STAGES * (1 + SFR) * SF);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + ACCS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + ACCS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* s_wg = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(full) + f4::BAR_BYTES);
    float* s_bias = s_wg + BN;
    const AbortCtx actx{abort_flag, p.error};

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int nk = (p.K + f4::KS - 1) / f4::KS, ntiles = p.tiles_m * p.tiles_n;

    if (tid == 0) {
        tma_prefetch_desc(&maps.w), tma_prefetch_desc(&maps.ws), tma_prefetch_desc(&maps.x), tma_prefetch_desc(&maps.xs);
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        for (int a = 0; a < ACCS; ++a) mbar_init(&acc_full[a], 1), mbar_init(&acc_empty[a], 2 * EW);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    // the peer's barriers must exist before anything of this CTA signals them
    cluster_arrive_release();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dependency_wait();
    grid_launch_dependents();

    if (warp == 0) {
        if (elect_lane()) {
            int it = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < ntiles; tile += npairs) {
                int tm, tn;
                fp4_tile(tile, p.tiles_m, p.tiles_n, tm, tn);
                const int row_a = tm * PAIR_M + (int)rank * BM, row_b = tn * BN + (int)rank * (BN / 2);
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (it >= STAGES && !mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, actx, kErrWaitEmpty)) {
                        ok = false;
                        break;
                    }
                    if (leader) mbar_expect_tx(&full[s], 2 * STAGE_BYTES);
                    const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
                    tma_load_2d_pair(sm + s * A_BYTES, &maps.x, bar, kb * f4::KSB, row_a);
                    tma_load_2d_pair(sm_b + s * B_BYTES, &maps.w, bar, kb * f4::KSB, row_b);
                    unsigned char* sf = sm_s + s * (1 + SFR) * SF;
                    tma_load_2d_pair(sf, &maps.xs, bar, kb * (SF / 8), row_a / 128);
                    tma_load_2d_pair(sf + SF, &maps.ws, bar, kb * (SF / 8), tn * SFR);
                }
            }
        }
    } else if (warp == 1) {
        if (leader && elect_lane()) {
            int it = 0, li = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < ntiles; tile += npairs, ++li) {
                const int as = li % ACCS;
                if (li >= ACCS && !mbar_wait_hot(&acc_empty[as], ((li / ACCS) - 1) & 1, actx, kErrWaitDFull)) break;
                tc_fence_after();
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait_hot(&full[s], (it / STAGES) & 1, actx, kErrWaitFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t sf = scale_desc(smem_u32(sm_s + s * (1 + SFR) * SF));
                    issue_stage<FORMAT, 2, PAIR_M, BN, SFR>(tmem + as * BN, make_sw128_kmajor_desc(smem_u32(sm + s * A_BYTES)),
                                                            make_sw128_kmajor_desc(smem_u32(sm_b + s * B_BYTES)),
                                                            tmem + ACCS * BN + s * sf_cols(FORMAT, BN), sf, sf + (uint64_t)(SF >> 4),
                                                            (p.K - kb * f4::KS + 63) / 64, kb == 0);
                    tc_commit_pair(&empty[s]);
                }
                if (ok) tc_commit_pair(&acc_full[as]);
            }
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2, et = tid - 64;  // (this thread among the epilogue's)
        constexpr int GROUPS = BN / 128;  // of 64 columns a warp
        unsigned char* stg = sm_o + (warp - 2) * STG_WARP_BYTES;
        const T* bias = static_cast<const T*>(p.bias);
        int li = 0;
        for (int tile = pair; tile < ntiles; tile += npairs, ++li) {
            const int as = li % ACCS;
            int tm, tn;
            fp4_tile(tile, p.tiles_m, p.tiles_n, tm, tn);
            // the tile's channel factors and bias (the warps meet on a barrier of their own: the last tile's are no longer read)
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int i = et; i < BN; i += 32 * EW) {
                const int n = tn * BN + i < p.N ? tn * BN + i : p.N - 1;
                s_wg[i] = p.wg ? p.wg[n] : 1.0f;
                s_bias[i] = bias ? to_f<T>(bias[n]) : 0.0f;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const int row0 = tm * PAIR_M + (int)rank * BM + q * 32, row = row0 + lane;
            const float gx = p.xg && row < p.M ? p.xg[row] : 1.0f;
            const bool staged = sizeof(T) == 2 && p.residual && p.vec;
            if (staged) request_residual(p, row0, tn * BN + half * GROUPS * 64, lane, stg);
            bool ok = true;
            if (lane == 0) ok = mbar_wait(&acc_full[as], (li / ACCS) & 1, actx, kErrWaitDFull);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) continue;  // (not out of the loop: the warps still meet at its barriers)
            tc_fence_after();
            // all of this warp's columns at once, then the accumulator goes back: with one accumulator the MMAs wait for this alone
            uint32_t v[GROUPS][64];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) tmem_ld64(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(as * BN + (half * GROUPS + g) * 64), v[g]);
            tc_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(&acc_empty[as]);
                else mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[as]), 0));
            }
            if (row0 >= p.M) continue;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int c0 = (half * GROUPS + g) * 64, col0 = tn * BN + c0;
                if (col0 >= p.N) continue;
                if (p.relu2) fp4_columns<FORMAT, T, 1>(p, maps.y, v[g], s_wg + c0, s_bias + c0, gx, row0, col0, lane, stg);
                else if (p.residual) fp4_columns<FORMAT, T, 2>(p, maps.y, v[g], s_wg + c0, s_bias + c0, gx, row0, col0, lane, stg);
                else fp4_columns<FORMAT, T, 0>(p, maps.y, v[g], s_wg + c0, s_bias + c0, gx, row0, col0, lane, stg);
                if (staged && g + 1 < GROUPS) request_residual(p, row0, col0 + 64, lane, stg);
            }
        }
        if (lane == 0) tma_store_wait_all();
    }
    // neither CTA may free its tensor memory or leave while the other can still touch its memory
    tc_fence_before();
    __syncthreads();
    cluster_arrive_release();
    cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, TMEM_COLS);
    }
}

// ---------------------------------------------------------------- host
// scale tiles as a matrix of 8-byte words, a row-tile a row; boxes of `box_rows` row tiles x one stage
static int make_tmap_scales(CUtensorMap* map, const void* base, int rows, int K, int format, int box_rows) {
    return make_tmap_2d(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 8, base, (uint64_t)(rows + 127) / 128, (uint64_t)fp4::k_tiles(K, format) * 64,
                        (uint32_t)box_rows, (uint32_t)f4::sf_bytes(format) / 8, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// CTAs that share the K range of a tile: as many as fit beside one another and keep two stages each.  us a call, 1 / 2 / 4 / 8, 16
// tokens: 768 -> 768 (three stages) 5.0 / 5.7 / - / -; 2560 -> 2560 7.0 / 6.6 / 6.1 / 9.9 (not all resident); 4096 -> 4096 8.7 / 7.6 / 6.7 /
// 13.9; 16384 -> 4096 21.8 / 14.8 / 12.0 / 21.0; 4096 -> 16384 9.1 / 14.0 / 20.6 / 38.2
static int stream_splits(int64_t tiles, int stages) {
    int splits = 1;
    while (splits < fs::MAX_SPLITS && 4 * splits <= stages && tiles * 2 * splits <= kSMs) splits *= 2;
    return splits;
}

template <int FORMAT, typename T, int BN, bool DEEP, bool FUSED = false>
static int launch_stream(const void* w, const void* ws, const void* xq, const void* xs, Fp4Args a, cudaStream_t st) {
    Fp4Maps m{};
    if (int e = make_tmap_2d(&m.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, a.N, a.K / 2, fs::BM, f4::KSB, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
    if (int e = make_tmap_scales(&m.ws, ws, a.N, a.K, FORMAT, 1)) return e;
    if constexpr (!FUSED) {
        if (int e = make_tmap_2d(&m.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xq, a.M, a.K / 2, BN, f4::KSB, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
        if (int e = make_tmap_scales(&m.xs, xs, a.M, a.K, FORMAT, 1)) return e;
    }
    auto kernel = fp4_stream_kernel<FORMAT, T, BN, DEEP, FUSED>;
    constexpr int smem = fs::smem_bytes(FORMAT, BN, DEEP, FUSED);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    RWKV7_REQUIRE(e == cudaSuccess, RWKV7_ERR_CUDA, "fp4_linear: %s", cudaGetErrorString(e));
    const int tn = (a.N + fs::BM - 1) / fs::BM, tm = (a.M + BN - 1) / BN;
    a.splits = DEEP ? stream_splits((int64_t)tn * tm, (a.K + f4::KS - 1) / f4::KS) : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tn, tm, a.splits);
    cfg.blockDim = dim3(fs::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = a.splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic_launch_ok(st) ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, m, a);
    return check_launch("fp4_stream_kernel");
}

template <int FORMAT, typename T, int BN>
static int launch_pair(const void* w, const void* ws, const void* xq, const void* xs, Fp4Args a, cudaStream_t st) {
    Fp4Maps m{};
    if (int e = make_tmap_2d(&m.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, a.N, a.K / 2, BN / 2, f4::KSB, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
    if (int e = make_tmap_2d(&m.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xq, a.M, a.K / 2, fp::BM, f4::KSB, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
    if (int e = make_tmap_scales(&m.ws, ws, a.N, a.K, FORMAT, fp::sfb_rows(BN))) return e;
    if (int e = make_tmap_scales(&m.xs, xs, a.M, a.K, FORMAT, 1)) return e;
    if (sizeof(T) == 2 && a.vec) {
        const CUtensorMapDataType dt = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;  // (bits are copied)
        if (int e = make_tmap_2d(&m.y, dt, (int)sizeof(T), a.y, a.M, a.N, 32, 64, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
    }
    auto kernel = fp4_pair_kernel<FORMAT, T, BN>;
    constexpr int smem = fp::smem_bytes(FORMAT, BN);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    RWKV7_REQUIRE(e == cudaSuccess, RWKV7_ERR_CUDA, "fp4_linear: %s", cudaGetErrorString(e));
    a.tiles_m = (a.M + fp::PAIR_M - 1) / fp::PAIR_M, a.tiles_n = (a.N + BN - 1) / BN;
    const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
    const int pairs = (int)(tiles < kSMs / 2 ? tiles : kSMs / 2);
    const cudaError_t l = launch_programmatic(kernel, dim3(2 * pairs), dim3(fp::THREADS), smem, st, m, a);
    RWKV7_REQUIRE(l == cudaSuccess, RWKV7_ERR_CUDA, "fp4_linear: %s", cudaGetErrorString(l));
    return check_launch("fp4_pair_kernel");
}

// Whether the product quantises its tokens itself, one launch less: few of them, a grid of one CTA an SM, a K range a CTA that fits.  Every CTA
// then quantises its range of K again, which is worth it while there is little of it: by tokens x stages.  us with the quantiser / without, weights out
// of memory, nvfp4: 1 x 4096 -> 16384 (16) 11.0 / 9.6, 1 x 10240 -> 2560 (10) 9.1 / 8.3, 4 x 4096 -> 4096 (16) 7.0 / 7.0, 4 x 768 -> 768 (12) 4.5 / 4.1, 8 x 768 -> 768 (24)
// 4.5 / 4.8, 2 x 4096 -> 16384 (32) 11.2 / 11.5; mxfp4, which needs no largest magnitude of the row: 1 x 4096 -> 16384 10.8 / 8.6, 4 x 16384 -> 4096 (64)
// 12.8 / 11.8, 4 x 4096 -> 16384 (64) 10.9 / 10.9, 8 x 2560 -> 10240 (80) 7.3 / 7.9.  A call costs the host 13.1 us instead of 15.7.
static bool quantises_itself(int M, int K, int N, int format) {
    const int tiles = (N + fs::BM - 1) / fs::BM, stages = (K + f4::KS - 1) / f4::KS, splits = stream_splits(tiles, stages);
    const int range = (stages + splits - 1) / splits;
    return M <= 16 && tiles <= kSMs && range <= fs::FUSED_STAGES && M * range <= (format == fp4::MX ? 64 : 16);
}

template <int FORMAT, typename T>
static int dispatch_fp4(const void* w, const void* ws, const void* xq, const void* xs, const Fp4Args& a, cudaStream_t st) {
    const int tiles = (a.N + fs::BM - 1) / fs::BM, stages = (a.K + f4::KS - 1) / f4::KS;
    // more tiles than SMs (an output head): two CTAs an SM, the start of one under the end of the other
    if (a.M <= 16) return tiles > kSMs ? launch_stream<FORMAT, T, 16, false>(w, ws, xq, xs, a, st) : launch_stream<FORMAT, T, 16, true>(w, ws, xq, xs, a, st);
    if (a.M <= 32) return tiles > kSMs ? launch_stream<FORMAT, T, 32, false>(w, ws, xq, xs, a, st) : launch_stream<FORMAT, T, 32, true>(w, ws, xq, xs, a, st);
    if (a.M <= 64 && tiles <= kSMs) return launch_stream<FORMAT, T, 64, true>(w, ws, xq, xs, a, st);
    const int64_t fit = kSMs / 2, tm = (a.M + fp::PAIR_M - 1) / fp::PAIR_M;
    const auto waves = [&](int bn) { return (tm * ((a.N + bn - 1) / bn) + fit - 1) / fit; };
    if (a.M <= 128) {
        // tenths of us: what a launch costs, and a stage of K of each wave
        const int64_t pair = (waves(128) * 27 < waves(256) * 30 ? 36 + waves(128) * stages * 27 / 10 : 39 + waves(256) * stages * 30 / 10);
        const int splits = stream_splits(tiles, stages);
        const int64_t stream = 20 + (tiles + kSMs - 1) / kSMs * ((splits > 1 ? 58 : 42) + stages / splits * 25 / 10);
        if (stream <= pair) return launch_stream<FORMAT, T, 128, true>(w, ws, xq, xs, a, st);
    }
    // a tile of half the channels takes two thirds of the time at best (its tokens are read as often, the way into shared memory bounds both) but
    // leaves fewer pairs idle; us of 128 / 256 channels: 512 x 4096 -> 4096 (one turn either way) 12.4 / 13.8, 512 x 16384 -> 4096 27.9 / 32.1, 1536 x 16384 ->
    // 4096 (three turns, two) 71.6 / 66.8, 1024 x 4096 -> 4096 (two, one) 18.1 / 15.9, 2048 x 4096 -> 16384 (14, 7) 78.3 / 64.9
    if (waves(128) * 2 < waves(256) * 3) return launch_pair<FORMAT, T, 128>(w, ws, xq, xs, a, st);
    return launch_pair<FORMAT, T, 256>(w, ws, xq, xs, a, st);
}

// Where the quantised tokens lie in the workspace: codes, scale tiles, row factors
struct Fp4Workspace {
    int64_t scales, row_scale, total;
    Fp4Workspace(int M, int K, int format) {
        auto up = [](int64_t v) { return (v + 127) / 128 * 128; };
        scales = up((int64_t)M * (K / 2));
        row_scale = scales + up(fp4::scale_bytes(M, K, format));
        total = row_scale + up(4ll * M);
    }
};

}  // namespace rwkv7

using namespace rwkv7;

extern "C" int64_t rwkv7_fp4_linear_workspace_bytes(int M, int K, int format) {
    if (M <= 0 || K <= 0 || K % 32 || (format != fp4::MX && format != fp4::NV)) return 0;
    return Fp4Workspace(M, K, format).total;
}

extern "C" int rwkv7_fp4_linear(const void* x, int64_t ldx, const void* w_packed, const void* w_scales, const float* w_row_scale,
                                const void* bias, const void* residual, void* y, void* workspace, int64_t workspace_bytes, int M, int K,
                                int N, int epilogue, int format, int dtype, void* stream) {
    RWKV7_REQUIRE(M > 0 && K > 0 && N > 0, RWKV7_ERR_INVALID, "fp4_linear: sizes must be positive");
    RWKV7_REQUIRE(format == fp4::MX || format == fp4::NV, RWKV7_ERR_INVALID, "fp4_linear: unknown format %d", format);
    RWKV7_REQUIRE(dtype >= RWKV7_F16 && dtype <= RWKV7_F32, RWKV7_ERR_INVALID, "fp4_linear: unknown dtype %d", dtype);
    RWKV7_REQUIRE(K % 32 == 0, RWKV7_ERR_UNSUPPORTED, "fp4_linear: K must be a multiple of 32 (got %d)", K);
    RWKV7_REQUIRE(x && w_packed && w_scales && y && workspace, RWKV7_ERR_INVALID, "fp4_linear: null pointer");
    RWKV7_REQUIRE(epilogue == RWKV7_EPI_NONE || epilogue == RWKV7_EPI_RELU2 || epilogue == RWKV7_EPI_ADD, RWKV7_ERR_INVALID,
                  "fp4_linear: unknown epilogue %d", epilogue);
    RWKV7_REQUIRE((epilogue == RWKV7_EPI_ADD) == (residual != nullptr), RWKV7_ERR_INVALID, "fp4_linear: the residual and its epilogue go together");
    RWKV7_REQUIRE(ldx >= K, RWKV7_ERR_INVALID, "fp4_linear: the row stride is shorter than a row");
    RWKV7_REQUIRE(aligned(x, 16) && (ldx * dtype_size(dtype)) % 16 == 0 && aligned(w_packed, 16) && aligned(w_scales, 16) && aligned(workspace, 128),
                  RWKV7_ERR_ALIGN, "fp4_linear: rows, weight and scales must be 16-byte aligned, the workspace 128-byte");
    const Fp4Workspace ws(M, K, format);
    RWKV7_REQUIRE(workspace_bytes >= ws.total, RWKV7_ERR_WORKSPACE, "fp4_linear: workspace of %lld bytes is smaller than the %lld required",
                  (long long)workspace_bytes, (long long)ws.total);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float* xg = reinterpret_cast<float*>(base + ws.row_scale);
    const bool fused = quantises_itself(M, K, N, format);
    if (!fused)
        if (int e = launch_fp4_quant(x, ldx, base, base + ws.scales, xg, M, K, format, dtype, st)) return e;
    Fp4Args a{};
    a.x = x, a.ldx = ldx;
    a.wg = w_row_scale, a.xg = format == fp4::NV ? xg : nullptr;
    a.bias = bias, a.residual = residual, a.y = y;
    a.M = M, a.N = N, a.K = K, a.relu2 = epilogue == RWKV7_EPI_RELU2;
    a.vec = N % 8 == 0 && aligned(y, 16) && (!residual || aligned(residual, 16));
    a.error = kernel_error_word();
    RWKV7_REQUIRE(a.error != nullptr, RWKV7_ERR_CUDA, "fp4_linear: cannot resolve the device error word");
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        if (fused)
            return format == fp4::MX ? launch_stream<fp4::MX, T, 16, true, true>(w_packed, w_scales, nullptr, nullptr, a, st)
                                     : launch_stream<fp4::NV, T, 16, true, true>(w_packed, w_scales, nullptr, nullptr, a, st);
        return format == fp4::MX ? dispatch_fp4<fp4::MX, T>(w_packed, w_scales, base, base + ws.scales, a, st)
                                 : dispatch_fp4<fp4::NV, T>(w_packed, w_scales, base, base + ws.scales, a, st);
    });
    return RWKV7_OK;
}
