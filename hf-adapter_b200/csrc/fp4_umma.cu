// Projection with both operands in microscaled 4-bit floating point (formats: fp4.cuh), on the block-scaled tensor cores:
//
//   y[m, n] = epilogue( gx[m] * gw[n] * sum_k q_x[m, k] s_x[m, k / block] q_w[n, k] s_w[n, k / block] )
//
// The weight is operand A (128 output channels a tile: the lanes of the accumulator), the tokens are operand B (the
// columns), so one kernel serves one token and thousands.  A stage of the ring holds 256 elements of K: codes by TMA in
// the 128-byte swizzle that the MMA reads, scale tiles by plain bulk copies (they lie in memory as tensor memory wants them).
// Warp 0 = producer, warp 1 = MMA issuer (copies a stage's scales to tensor memory, then issues its MMAs of 64 k; both
// run in issue order), warps 2-5 = epilogue.  All waits are bounded (umma.cuh).
#include "fp4.cuh"
#include "umma.cuh"

namespace rwkv7 {
namespace f4 {
constexpr int BM = 128, BKB = 128, THREADS = 192;  // channels a tile, bytes (256 elements) of K a stage
constexpr int A_BYTES = BM * BKB;
constexpr int tiles_per_stage(int format) { return format == fp4::MX ? 2 : 4; }  // scale tiles of 128 rows
constexpr int sf_rows(int bn) { return (bn + 127) / 128; }
constexpr int sf_bytes(int format) { return tiles_per_stage(format) * fp4::SCALE_TILE_BYTES; }
constexpr int stage_bytes(int format, int bn) { return A_BYTES + bn * BKB + (1 + sf_rows(bn)) * sf_bytes(format); }
constexpr int stages(int bn) { return bn == 256 ? 4 : 6; }
constexpr int BAR_BYTES = 1024;
constexpr int smem_bytes(int format, int bn) { return stages(bn) * stage_bytes(format, bn) + BAR_BYTES + bn * 4 + 1024; }
// tensor memory: the accumulator, then per stage the scales of A (4 columns a tile) and of B
constexpr int sf_cols(int format, int bn) { return tiles_per_stage(format) * 4 * (1 + sf_rows(bn)); }
constexpr int tmem_cols(int format, int bn) {
    int need = bn + stages(bn) * sf_cols(format, bn), c = 32;
    while (c < need) c *= 2;
    return c;
}
}  // namespace f4

struct Fp4Args {
    const uint8_t *ws, *xs;        // scale tiles of the weight and the tokens
    const float *wg, *xg;          // row factors (nvfp4; NULL = 1)
    const void *bias, *residual;
    void* y;
    int M, N, K;
    int relu2;
    unsigned int* error;
};

// Instruction descriptor of the block-scaled 4-bit kinds: E2M1 operands (1), scale type (0 = E4M3, 1 = E8M0), and which
// byte of a scale word the first block of this K step has (0, or 2 for the second half of a word with two scales a step).
__host__ __device__ constexpr uint32_t fp4_idesc(int M, int N, int e8m0, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)e8m0 << 23) | ((uint32_t)(M >> 7) << 27) | (sf_id << 29);
}
template <int FORMAT>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (FORMAT == fp4::MX)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// One scale tile (32 rows of 16 bytes, 8-row groups 128 bytes apart) to four columns, repeated in the four lane quarters
__device__ __forceinline__ void copy_scale_tile(uint32_t taddr, uint32_t smem_addr) {
    uint64_t d = (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint64_t* bar, uint32_t bytes) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <int FORMAT, typename T, int BN>
__global__ void __launch_bounds__(f4::THREADS, 1)
fp4_umma_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Fp4Args p) {
    using namespace f4;
    constexpr int STAGES = stages(BN), STAGE_BYTES = stage_bytes(FORMAT, BN), TPS = tiles_per_stage(FORMAT), SFR = sf_rows(BN);
    constexpr int SFB_BYTES = sf_bytes(FORMAT), TMEM_COLS = tmem_cols(FORMAT, BN), SF_COLS = sf_cols(FORMAT, BN);
    static_assert(BN + STAGES * SF_COLS <= TMEM_COLS && TMEM_COLS <= 512, "tensor memory");
    extern __shared__ unsigned char smem_unaligned[];
    unsigned char* sm = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    // [A of all stages][B of all stages][scales of all stages][barriers][row factors of the tokens]
    unsigned char* sm_b = sm + STAGES * A_BYTES;
    unsigned char* sm_s = sm_b + STAGES * BN * BKB;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + STAGES * STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* s_xg = reinterpret_cast<float*>(sm + STAGES * STAGE_BYTES + BAR_BYTES);
    const AbortCtx actx{abort_flag, p.error};

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n0 = blockIdx.x * BM, m0 = blockIdx.y * BN;
    const int nk = (p.K + 2 * BKB - 1) / (2 * BKB);
    const int ktiles = fp4::k_tiles(p.K, FORMAT);

    if (tid == 0) {
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        mbar_init(acc_full, 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
    for (int i = tid; i < BN; i += THREADS) s_xg[i] = p.xg && m0 + i < p.M ? p.xg[m0 + i] : 1.0f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            const int x_tiles = (p.M + 127) / 128, rt = m0 / 128;
            const int sfb_rows = x_tiles - rt < SFR ? x_tiles - rt : SFR;  // scale row-tiles that exist
            for (int kb = 0; kb < nk; ++kb) {
                const int s = kb % STAGES;
                if (kb >= STAGES && !mbar_wait(&empty[s], ((kb / STAGES) - 1) & 1, actx, kErrWaitEmpty)) break;
                const int kt = kb * TPS, live = ktiles - kt < TPS ? ktiles - kt : TPS;
                const uint32_t sf = live * fp4::SCALE_TILE_BYTES;
                mbar_expect_tx(&full[s], A_BYTES + BN * BKB + sf * (1 + sfb_rows));
                tma_load_2d(sm + s * A_BYTES, &tm_w, &full[s], kb * BKB, n0);
                tma_load_2d(sm_b + s * BN * BKB, &tm_x, &full[s], kb * BKB, m0);
                unsigned char* sf_dst = sm_s + s * (1 + SFR) * SFB_BYTES;
                bulk_load(sf_dst, p.ws + ((size_t)blockIdx.x * ktiles + kt) * fp4::SCALE_TILE_BYTES, &full[s], sf);
                for (int r = 0; r < sfb_rows; ++r)
                    bulk_load(sf_dst + (1 + r) * SFB_BYTES, p.xs + ((size_t)(rt + r) * ktiles + kt) * fp4::SCALE_TILE_BYTES, &full[s], sf);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            for (int kb = 0; kb < nk; ++kb) {
                const int s = kb % STAGES;
                if (!mbar_wait_hot(&full[s], (kb / STAGES) & 1, actx, kErrWaitFull)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const int steps = (p.K - kb * 256 + 63) / 64 < 4 ? (p.K - kb * 256 + 63) / 64 : 4;  // of 64 elements
                const uint32_t sfa = tmem + BN + s * SF_COLS, sfb = sfa + TPS * 4;
                const uint32_t sf_src = smem_u32(sm_s + s * (1 + SFR) * SFB_BYTES);
                for (int t = 0; t < TPS; ++t) {
                    if (t * 4 / TPS >= steps) break;
                    copy_scale_tile(sfa + 4 * t, sf_src + t * fp4::SCALE_TILE_BYTES);
#pragma unroll
                    for (int r = 0; r < SFR; ++r)
                        copy_scale_tile(sfb + 4 * (t * SFR + r), sf_src + (1 + r) * SFB_BYTES + t * fp4::SCALE_TILE_BYTES);
                }
                const uint64_t da = make_sw128_kmajor_desc(smem_u32(sm + s * A_BYTES));
                const uint64_t db = make_sw128_kmajor_desc(smem_u32(sm_b + s * BN * BKB));
                for (int j = 0; j < steps; ++j) {
                    const int t = FORMAT == fp4::MX ? j >> 1 : j;
                    const uint32_t id = FORMAT == fp4::MX && (j & 1) ? fp4_idesc(BM, BN, 1, 2) : fp4_idesc(BM, BN, FORMAT == fp4::MX, 0);
                    umma_fp4<FORMAT>(tmem, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), id, sfa + 4 * t, sfb + 4 * SFR * t,
                                     kb > 0 || j > 0);
                }
                tc_commit(&empty[s]);
            }
            if (ok) tc_commit(acc_full);
        }
    } else {
        const int q = warp & 3, n = n0 + q * 32 + lane;
        bool ok = true;
        if (lane == 0) ok = mbar_wait(acc_full, 0, actx, kErrWaitDFull);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (ok) {
            tc_fence_after();
            const float gw = p.wg && n < p.N ? p.wg[n] : 1.0f;
            const float b = p.bias && n < p.N ? to_f<T>(static_cast<const T*>(p.bias)[n]) : 0.0f;
#pragma unroll 1
            for (int c = 0; c < BN; c += 16) {
                if (m0 + c >= p.M) break;
                uint32_t v[16];
                tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
                tc_wait_ld();
                if (n < p.N) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int m = m0 + c + i;
                        if (m < p.M) {
                            float y = __uint_as_float(v[i]) * (gw * s_xg[c + i]) + b;
                            if (p.relu2) y = y > 0.0f ? y * y : y != y ? y : 0.0f;
                            if (p.residual) y += to_f<T>(static_cast<const T*>(p.residual)[(size_t)m * p.N + n]);
                            static_cast<T*>(p.y)[(size_t)m * p.N + n] = from_f<T>(y);
                        }
                    }
                }
            }
            tc_fence_before();
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

template <int FORMAT, typename T, int BN>
static int launch_fp4(const void* w, const void* xq, const Fp4Args& a, cudaStream_t st) {
    CUtensorMap tm_w, tm_x;
    if (int e = make_tmap_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, a.N, a.K / 2, f4::BM, f4::BKB, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
    if (int e = make_tmap_2d(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xq, a.M, a.K / 2, BN, f4::BKB, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
    auto kernel = fp4_umma_kernel<FORMAT, T, BN>;
    constexpr int smem = f4::smem_bytes(FORMAT, BN);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    RWKV7_REQUIRE(e == cudaSuccess, RWKV7_ERR_CUDA, "fp4_linear: %s", cudaGetErrorString(e));
    kernel<<<dim3((a.N + f4::BM - 1) / f4::BM, (a.M + BN - 1) / BN), f4::THREADS, smem, st>>>(tm_w, tm_x, a);
    return check_launch("fp4_umma_kernel");
}

// (a tile narrower than 128 tokens is used for a first tile alone: the scales of its tokens begin in the first column of their tile)
template <int FORMAT, typename T>
static int dispatch_fp4(const void* w, const void* xq, const Fp4Args& a, cudaStream_t st) {
    if (a.M <= 16) return launch_fp4<FORMAT, T, 16>(w, xq, a, st);
    if (a.M <= 64) return launch_fp4<FORMAT, T, 64>(w, xq, a, st);
    if (a.M <= 512) return launch_fp4<FORMAT, T, 128>(w, xq, a, st);
    return launch_fp4<FORMAT, T, 256>(w, xq, a, st);
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
    if (int e = launch_fp4_quant(x, ldx, base, base + ws.scales, xg, M, K, format, dtype, st)) return e;
    Fp4Args a{};
    a.ws = static_cast<const uint8_t*>(w_scales), a.xs = base + ws.scales;
    a.wg = w_row_scale, a.xg = format == fp4::NV ? xg : nullptr;
    a.bias = bias, a.residual = residual, a.y = y;
    a.M = M, a.N = N, a.K = K, a.relu2 = epilogue == RWKV7_EPI_RELU2;
    a.error = kernel_error_word();
    RWKV7_REQUIRE(a.error != nullptr, RWKV7_ERR_CUDA, "fp4_linear: cannot resolve the device error word");
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        return format == fp4::MX ? dispatch_fp4<fp4::MX, T>(w_packed, base, a, st) : dispatch_fp4<fp4::NV, T>(w_packed, base, a, st);
    });
    return RWKV7_OK;
}
