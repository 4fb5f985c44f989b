// Rows to microscaled 4-bit floating point and back (formats: fp4.cuh).
//
//   mxfp4: byte = max(E - 2, 0), E the biased exponent of the block's largest magnitude (so 2^(floor(log2 amax) - 2)),
//          code = e2m1(x * 2^(127 - byte)); magnitudes in (6, 8) units saturate at 6.
//   nvfp4: g = 2^(floor(log2 amax of the row) - 10) (1 for a row of zeros), s = e4m3(amax of the block / g / 6),
//          code = e2m1(x / g / s), 0 where s is 0.  amax / g / 6 stays below 342, inside E4M3's 448.
//
// Every rounding is to nearest, ties to even: powers of two divide exactly; x / s is formed as a product with 1 / s and one
// correction step, which is the correctly rounded quotient; a sixth is taken as the product with the fp32 nearest to 1 / 6,
// 2^-25 off, so six times a number of few bits gives that number.  For fp16 / bf16 input a tie is therefore met exactly or missed
// by 2^-12 at least; fp32 input can round the other way where the quotient is within 2^-23 of one.
// A block with an element that is not finite gets a NaN scale; the row's largest magnitude is taken over the finite
// ones.
#include <cuda_fp8.h>

#include "fp4.cuh"

namespace rwkv7 {
using namespace fp4;

// eight codes, element 0 in the lowest nibble
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    uint32_t d;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(d) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}

// values of two codes (one byte)
__device__ __forceinline__ float2 unpack2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 a, z;\n\tmov.b32 {a, z, z, z}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return byte == 255 ? __int_as_float(0x7fffffff) : byte ? __int_as_float(byte << 23) : __int_as_float(1 << 22);
}

// the largest finite magnitude of 16 elements, and whether all are finite
__device__ __forceinline__ float finite_amax(const float (&v)[16], bool& finite) {
    float m = 0.0f;
    finite = true;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float a = fabsf(v[i]);
        const bool ok = a < INFINITY;  // false for NaN too
        finite &= ok;
        m = fmaxf(m, ok ? a : 0.0f);
    }
    return m;
}

template <typename T> __device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float o[8];
        load8<T>(p + 8 * h, o);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * h + i] = o[i];
    }
}

// A CTA a row, 16 elements a thread and pass.  Rows beyond R pad the last scale tile with zeros.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(256) fp4_quant_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ packed,
                                                        uint8_t* __restrict__ scales, float* __restrict__ row_scale, int R, int K) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const int ktiles = k_tiles(K, FORMAT), pieces = K / 16;
    const int padded = ktiles * SCALE_TILE_BLOCKS * block_of(FORMAT) / 16;  // pieces that the scale tiles cover
    const int lane = threadIdx.x & 31;
    if (row >= R) {
        for (int t = threadIdx.x; t < ktiles; t += blockDim.x) *reinterpret_cast<uint32_t*>(scales + scale_word(row, t, ktiles)) = 0;
        return;
    }
    const T* xr = x + row * ldx;
    float inv_g = 1.0f;
    if (FORMAT == NV) {
        float m = 0.0f;
        for (int p = threadIdx.x; p < pieces; p += blockDim.x) {
            float v[16];
            bool finite;
            load16<T>(xr + 16 * p, v);
            m = fmaxf(m, finite_amax(v, finite));
        }
        m = block_max(m, red);
        const int e = max(__float_as_int(m) >> 23, 1);  // biased exponent; subnormal magnitudes count as the smallest normal
        const int ge = m > 0.0f ? max(e - 10, 1) : 127;
        inv_g = __int_as_float((254 - ge) << 23);
        if (threadIdx.x == 0) row_scale[row] = __int_as_float(ge << 23);
    }
    // whole warps stay in the loop for the shuffles
    for (int p0 = threadIdx.x - lane; p0 < padded; p0 += blockDim.x) {
        const int p = p0 + lane;
        const bool live = p < pieces;
        float v[16];
        if (live) load16<T>(xr + 16 * p, v);
        else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.0f;
        }
        bool finite;
        float m = finite_amax(v, finite);
        uint32_t byte;
        float mult;
        if (FORMAT == MX) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            finite = __shfl_xor_sync(0xffffffffu, (int)finite, 1) && finite;
            byte = max((__float_as_int(m) >> 23) - 2, 0);
            mult = __int_as_float((254 - byte) << 23);  // 2^(127 - byte); byte <= 252
            if (!finite) byte = 255;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= mult;
        } else {
            byte = __nv_cvt_float_to_fp8(m * inv_g * (1.0f / 6.0f), __NV_SATFINITE, __NV_E4M3);
            const float s = e4m3_value(byte);
            const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
            if (!finite) byte = 0x7f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float u = v[i] * inv_g, q = u * inv;
                v[i] = fmaf(fmaf(-q, s, u), inv, q);
            }
        }
        if (live) {
            float lo[8], hi[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[i] = v[i], hi[i] = v[8 + i];
            *reinterpret_cast<uint2*>(packed + row * (K / 2) + 8 * p) = make_uint2(pack8(lo), pack8(hi));
        } else {
            byte = 0;
        }
        // four scales to one word: blocks lie one (nvfp4) or two (mxfp4) lanes apart
        constexpr int STEP = block_of(FORMAT) / 16;
        uint32_t word = byte;
#pragma unroll
        for (int i = 1; i < 4; ++i) word |= __shfl_down_sync(0xffffffffu, byte, i * STEP) << (8 * i);
        if (lane % (4 * STEP) == 0 && p < padded) *reinterpret_cast<uint32_t*>(scales + scale_word(row, p / (4 * STEP), ktiles)) = word;
    }
}

template <typename T, int FORMAT>
__global__ void __launch_bounds__(256) fp4_dequant_kernel(const uint8_t* __restrict__ packed, const uint8_t* __restrict__ scales,
                                                          const float* __restrict__ row_scale, T* __restrict__ out, int64_t total, int K) {
    const int pieces = K / 16, ktiles = k_tiles(K, FORMAT);
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / pieces;
        const int p = (int)(i - row * pieces);
        const int block = FORMAT == MX ? p >> 1 : p;
        const uint32_t byte = scales[scale_word(row, block >> 2, ktiles) + (block & 3)];
        const float s = FORMAT == MX ? e8m0_value(byte) : e4m3_value(byte);
        const float g = FORMAT == MX || row_scale == nullptr ? 1.0f : row_scale[row];
        const uint2 c = *reinterpret_cast<const uint2*>(packed + i * 8);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t w = h ? c.y : c.x;
            float o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = unpack2((w >> (8 * j)) & 255);
                o[2 * j] = f.x * s * g, o[2 * j + 1] = f.y * s * g;
            }
            store8<T>(out + i * 16 + 8 * h, o);
        }
    }
}

template <typename T, int FORMAT>
static int quant(const void* x, int64_t ldx, uint8_t* packed, uint8_t* scales, float* row_scale, int rows, int K, cudaStream_t st) {
    const int ktiles = k_tiles(K, FORMAT);
    const int pieces = ktiles * SCALE_TILE_BLOCKS * block_of(FORMAT) / 16;
    const int threads = pieces >= 256 ? 256 : (pieces + 31) / 32 * 32;
    const int64_t grid = ((int64_t)rows + SCALE_TILE_ROWS - 1) / SCALE_TILE_ROWS * SCALE_TILE_ROWS;
    fp4_quant_kernel<T, FORMAT><<<(unsigned)grid, threads, 0, st>>>(static_cast<const T*>(x), ldx, packed, scales, row_scale, rows, K);
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
    RWKV7_REQUIRE(packed && scales && out, RWKV7_ERR_INVALID, "fp4_dequant: null pointer");
    RWKV7_REQUIRE(aligned(packed, 16) && aligned(scales, 16) && aligned(out, 16), RWKV7_ERR_ALIGN, "fp4_dequant: tensors must be 16-byte aligned");
    const int64_t total = (int64_t)rows * (K / 16);
    const unsigned grid = (unsigned)((total + 255) / 256 < 16 * kSMs ? (total + 255) / 256 : 16 * kSMs);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        auto kernel = format == MX ? fp4_dequant_kernel<T, MX> : fp4_dequant_kernel<T, NV>;
        kernel<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(packed), static_cast<const uint8_t*>(scales), row_scale,
                                     static_cast<T*>(out), total, K);
    });
    return check_launch("fp4_dequant_kernel");
}
