// Rows to microscaled 4-bit floating point and back (formats: fp4.cuh).
//
//   mxfp4: byte = max(E - 2, 0), E the biased exponent of the block's largest magnitude (so 2^(floor(log2 amax) - 2)),
//          code = e2m1(x * 2^(127 - byte)); magnitudes in (6, 8) units saturate at 6.
//   nvfp4: g = 2^(floor(log2 amax of the row) - 10) (1 for a row of zeros), s = e4m3(amax of the block / g / 6),
//          code = e2m1(x / g / s), 0 where s is 0.  amax / g / 6 stays below 342, inside E4M3's 448.
//
// Every rounding is to nearest, ties to even: powers of two divide exactly; x / s is formed as a product with 1 / s and, for fp32,
// one correction step, which makes it the correctly rounded quotient, for 16 bits rounded to steps of 2^-17 instead; a sixth is
// taken as the product with the fp32 nearest to 1 / 6, 2^-25 off, so six times a number of few bits gives that number.  For
// fp16 / bf16 input a tie is therefore met exactly or missed by 2^-12 at least; fp32 input can round the other way where the
// quotient is within 2^-23 of one.
// A block with an element that is not finite gets a NaN scale; the row's largest magnitude is taken over the finite
// ones.
#include "fp4_encode.cuh"

namespace rwkv7 {
using namespace fp4;

// values of two codes (one byte)
__device__ __forceinline__ float2 unpack2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 a, z;\n\tmov.b32 {a, z, z, z}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}

__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return byte == 255 ? __int_as_float(0x7fffffff) : byte ? __int_as_float(byte << 23) : __int_as_float(1 << 22);
}

// `team` threads a row, P pieces of 16 elements a thread, read once and kept (P = 0: read again for the codes).  Rows beyond R
// pad the last scale tile with zeros.  Bound by the memory for many rows, where nvfp4 also waits for the row's maximum before its first code: 8192 x 4096
// bf16 (67 MB in, 18 to 19 out) mxfp4 14.8 us = 5.7 TB/s, nvfp4 18.8 us = 4.6 TB/s; by the launch for few: 1 x 768 1.3 and 1.8 us, 64 x 4096 1.7 and 2.1.
template <typename T, int FORMAT, int P>
__global__ void __launch_bounds__(256) fp4_quant_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ packed,
                                                        uint8_t* __restrict__ scales, float* __restrict__ row_scale, int R, int K, int team) {
    __shared__ float red[8];
    const int at = threadIdx.x % team, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / team) + threadIdx.x / team;
    const int ktiles = k_tiles(K, FORMAT), pieces = row < R ? K / 16 : 0;
    const int padded = ktiles * SCALE_TILE_BLOCKS * block_of(FORMAT) / 16;  // pieces that the scale tiles cover
    grid_dependency_wait();
    grid_launch_dependents();
    const T* xr = x + row * ldx;
    Piece<T> kept[P ? P : 1];
    float most[P ? P : 1];
    if constexpr (P > 0) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int p = at + i * team;
            kept[i] = Piece<T>{};
            if (p < pieces) kept[i] = load_piece<T>(xr + 16 * p);
        }
    }
    int ge = 127;
    if constexpr (FORMAT == NV) {
        float m = 0.0f;
        if constexpr (P > 0) {
#pragma unroll
            for (int i = 0; i < P; ++i) most[i] = piece_amax(kept[i]), m = fmaxf(m, finite_amax(kept[i], most[i]));
        } else {
            for (int p = at; p < pieces; p += team) {
                const Piece<T> one = load_piece<T>(xr + 16 * p);
                m = fmaxf(m, finite_amax(one, piece_amax(one)));
            }
        }
        m = group_max<32>(m);
        if (team > 32) {
            if (lane == 0) red[threadIdx.x >> 5] = m;
            __syncthreads();
            for (int w = threadIdx.x / team * (team / 32), n = team / 32; n > 0; ++w, --n) m = fmaxf(m, red[w]);
        }
        const int e = max(__float_as_int(m) >> 23, 1);  // biased exponent; subnormal magnitudes count as the smallest normal
        ge = m > 0.0f ? max(e - 10, 1) : 127;
        if (at == 0 && row < R) row_scale[row] = __int_as_float(ge << 23);
    }
    const auto put = [&](const Piece<T>& piece, float m, int p) {
        uint2 codes;
        uint32_t byte = encode_piece<T, FORMAT>(piece, m, ge, codes);
        if (p < pieces) *reinterpret_cast<uint2*>(packed + row * (K / 2) + 8 * p) = codes;
        else byte = 0;
        // four scales to one word: blocks lie one (nvfp4) or two (mxfp4) lanes apart
        constexpr int STEP = block_of(FORMAT) / 16;
        uint32_t word = byte | __shfl_down_sync(0xffffffffu, byte, STEP) << 8;
        word |= __shfl_down_sync(0xffffffffu, word, 2 * STEP) << 16;
        if (lane % (4 * STEP) == 0 && p < padded) *reinterpret_cast<uint32_t*>(scales + scale_word(row, p / (4 * STEP), ktiles)) = word;
    };
    if constexpr (P > 0) {
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (at - lane + i * team < padded) put(kept[i], FORMAT == NV ? most[i] : piece_amax(kept[i]), at + i * team);  // (whole warps, for the shuffles)
    } else {
        for (int p0 = at - lane; p0 < padded; p0 += team) {
            const int p = p0 + lane;
            Piece<T> one{};
            if (p < pieces) one = load_piece<T>(xr + 16 * p);
            put(one, piece_amax(one), p);
        }
    }
}

// 16 bytes of values a thread, four of them a turn; INDEX wide enough to count them.  Bound by the memory: 8192 x 4096 to bf16 (85 MB) 16.2 us
// (mxfp4) and 17.5 us (nvfp4) = 5.2 and 4.9 TB/s.
template <typename T, int FORMAT, typename INDEX>
__global__ void __launch_bounds__(256) fp4_dequant_kernel(const uint8_t* __restrict__ packed, const uint8_t* __restrict__ scales,
                                                          const float* __restrict__ row_scale, T* __restrict__ out, INDEX total, int K) {
    constexpr int E = 16 / sizeof(T);  // elements
    const unsigned pieces = K / E;
    const int ktiles = k_tiles(K, FORMAT);
    grid_dependency_wait();
    grid_launch_dependents();
    const INDEX stride = (INDEX)gridDim.x * blockDim.x;
    for (INDEX i0 = (INDEX)blockIdx.x * blockDim.x + threadIdx.x; i0 < total; i0 += 4 * stride) {
        uint32_t code[4], byte[4];
        float g[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const INDEX i = i0 + u * stride;
            if (i < total) {
                const INDEX row = i / pieces;
                const int block = (int)(i - row * pieces) * E / block_of(FORMAT);
                code[u] = E == 8 ? *reinterpret_cast<const uint32_t*>(packed + (int64_t)i * (E / 2)) : *reinterpret_cast<const uint16_t*>(packed + (int64_t)i * (E / 2));
                byte[u] = scales[scale_word((int64_t)row, block >> 2, ktiles) + (block & 3)];
                g[u] = FORMAT == MX || row_scale == nullptr ? 1.0f : row_scale[row];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const INDEX i = i0 + u * stride;
            if (i < total) {
                const float s = FORMAT == MX ? e8m0_value(byte[u]) : e4m3_value(byte[u]);
                float o[E];
#pragma unroll
                for (int j = 0; j < E / 2; ++j) {
                    const float2 f = unpack2((code[u] >> (8 * j)) & 255);
                    o[2 * j] = f.x * s * g[u], o[2 * j + 1] = f.y * s * g[u];
                }
                if constexpr (E == 8) store8<T>(out + (int64_t)i * E, o);
                else store4<T>(out + (int64_t)i * E, o);
            }
        }
    }
}

template <typename T, int FORMAT>
static int quant(const void* x, int64_t ldx, uint8_t* packed, uint8_t* scales, float* row_scale, int rows, int K, cudaStream_t st) {
    const int ktiles = k_tiles(K, FORMAT);
    const int pieces = ktiles * SCALE_TILE_BLOCKS * block_of(FORMAT) / 16;
    // Few rows: a piece a thread, for the shortest way.  Many rows: four, and several rows a CTA.  us with one / four, nvfp4: 1 x 4096 2.1 / 3.2, 512 x 4096
    // 3.4 / 3.8, 1024 x 4096 4.6 / 4.6 (mxfp4 3.0 / 3.4), 8192 x 4096 22.6 / 19.2, 8192 x 768 6.7 / 5.4; one row a CTA there 9.5.
    const int per = rows >= 2048 ? 4 : 1;
    int team = 32;
    while (team < 256 && team * per < pieces) team *= 2;
    const int threads = rows >= 2048 ? 256 : team;
    const int64_t all = ((int64_t)rows + SCALE_TILE_ROWS - 1) / SCALE_TILE_ROWS * SCALE_TILE_ROWS, grid = all / (threads / team);
    auto kernel = pieces <= team ? fp4_quant_kernel<T, FORMAT, 1> : pieces <= 2 * team ? fp4_quant_kernel<T, FORMAT, 2>
                  : pieces <= 4 * team ? fp4_quant_kernel<T, FORMAT, 4> : fp4_quant_kernel<T, FORMAT, 0>;
    const cudaError_t e = launch_programmatic(kernel, dim3((unsigned)grid), dim3(threads), 0, st, static_cast<const T*>(x), ldx, packed, scales,
                                              row_scale, rows, K, team);
    RWKV7_REQUIRE(e == cudaSuccess, RWKV7_ERR_CUDA, "fp4_quant: %s", cudaGetErrorString(e));
    return check_launch("fp4_quant_kernel");
}

int launch_fp4_quant(const void* x, int64_t ldx, uint8_t* packed, uint8_t* scales, float* row_scale, int rows, int K, int format,
                     int dtype, cudaStream_t st) {
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        return format == MX ? quant<T, MX>(x, ldx, packed, scales, row_scale, rows, K, st)
                            : quant<T, NV>(x, ldx, packed, scales, row_scale, rows, K, st);
    });
    return RWKV7_OK;
}

}  // namespace rwkv7

using namespace rwkv7;

extern "C" int64_t rwkv7_fp4_scale_bytes(int rows, int K, int format) {
    if (rows <= 0 || K <= 0 || K % 32 || (format != MX && format != NV)) return 0;
    return fp4::scale_bytes(rows, K, format);
}

extern "C" int rwkv7_fp4_quant(const void* x, int64_t ldx, void* packed, void* scales, float* row_scale, int rows, int K, int format,
                               int dtype, void* stream) {
    RWKV7_REQUIRE(rows > 0 && K > 0, RWKV7_ERR_INVALID, "fp4_quant: sizes must be positive");
    RWKV7_REQUIRE(format == MX || format == NV, RWKV7_ERR_INVALID, "fp4_quant: unknown format %d", format);
    RWKV7_REQUIRE(K % 32 == 0, RWKV7_ERR_UNSUPPORTED, "fp4_quant: K must be a multiple of 32 (got %d)", K);
    RWKV7_REQUIRE(dtype >= RWKV7_F16 && dtype <= RWKV7_F32, RWKV7_ERR_INVALID, "fp4_quant: unknown dtype %d", dtype);
    RWKV7_REQUIRE(x && packed && scales && (row_scale || format == MX), RWKV7_ERR_INVALID, "fp4_quant: null pointer");
    RWKV7_REQUIRE(ldx >= K, RWKV7_ERR_INVALID, "fp4_quant: the row stride is shorter than a row");
    RWKV7_REQUIRE(aligned(x, 16) && (ldx * dtype_size(dtype)) % 16 == 0 && aligned(packed, 16) && aligned(scales, 16), RWKV7_ERR_ALIGN,
                  "fp4_quant: rows must be 16-byte aligned");
    return launch_fp4_quant(x, ldx, static_cast<uint8_t*>(packed), static_cast<uint8_t*>(scales), row_scale, rows, K, format, dtype,
                            static_cast<cudaStream_t>(stream));
}

extern "C" int rwkv7_fp4_dequant(const void* packed, const void* scales, const float* row_scale, void* out, int rows, int K, int format,
                                 int dtype, void* stream) {
    RWKV7_REQUIRE(rows > 0 && K > 0, RWKV7_ERR_INVALID, "fp4_dequant: sizes must be positive");
    RWKV7_REQUIRE(format == MX || format == NV, RWKV7_ERR_INVALID, "fp4_dequant: unknown format %d", format);
    RWKV7_REQUIRE(K % 32 == 0, RWKV7_ERR_UNSUPPORTED, "fp4_dequant: K must be a multiple of 32 (got %d)", K);
    RWKV7_REQUIRE(dtype >= RWKV7_F16 && dtype <= RWKV7_F32, RWKV7_ERR_INVALID, "fp4_dequant: unknown dtype %d", dtype);
    RWKV7_REQUIRE(packed && scales && out, RWKV7_ERR_INVALID, "fp4_dequant: null pointer");
    RWKV7_REQUIRE(aligned(packed, 16) && aligned(scales, 16) && aligned(out, 16), RWKV7_ERR_ALIGN, "fp4_dequant: tensors must be 16-byte aligned");
    const int64_t total = (int64_t)rows * (K / (16 / (int)dtype_size(dtype))), turns = (total + 1023) / 1024;
    const unsigned grid = (unsigned)(turns < 8 * kSMs ? turns : 8 * kSMs);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const auto *c = static_cast<const uint8_t*>(packed), *s = static_cast<const uint8_t*>(scales);
    cudaError_t e = cudaSuccess;
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        T* o = static_cast<T*>(out);
        if (total < (1ll << 31)) {  // (the turns after the last one stay inside 32 bits too)
            auto kernel = format == MX ? fp4_dequant_kernel<T, MX, uint32_t> : fp4_dequant_kernel<T, NV, uint32_t>;
            e = launch_programmatic(kernel, dim3(grid), dim3(256), 0, st, c, s, row_scale, o, (uint32_t)total, K);
        } else {
            auto kernel = format == MX ? fp4_dequant_kernel<T, MX, int64_t> : fp4_dequant_kernel<T, NV, int64_t>;
            e = launch_programmatic(kernel, dim3(grid), dim3(256), 0, st, c, s, row_scale, o, total, K);
        }
    });
    RWKV7_REQUIRE(e == cudaSuccess, RWKV7_ERR_CUDA, "fp4_dequant: %s", cudaGetErrorString(e));
    return check_launch("fp4_dequant_kernel");
}
