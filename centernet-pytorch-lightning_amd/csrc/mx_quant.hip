// Quantisation to block-scaled 8- / 4-bit floating point and back (formats: mx_common.h).
//
// Both directions stream: a thread owns eight consecutive channels (16 or 32 bytes of the tensor), the four threads of a quad own one
// block, so the block's maximum is two cross-lane moves and nothing is staged.  Chunks of 8 are numbered through the padded rows
// (4 per block), which keeps every store of codes aligned and contiguous over the wave.
// Bound by memory: 1048576 x 64 bf16 to e4m3 38 us (203 MB, 5.3 TB/s) and back 30 us (what was just written is still in the memory-side
// cache); 32 x 512 2.6 us, a launch.
#include "mx_common.h"

// U: chunks a thread has in flight; FULL: C is a multiple of 8
template <typename T, int FMT, bool SIGNS, int U, bool FULL>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, const T* __restrict__ sg, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, uint8_t* __restrict__ signs, int64_t chunks, int C,
                                                          MxDiv cpr) {
    const int64_t base = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = base / cpr.d;                                   // (uniform: one 64-bit division per workgroup)
    const uint32_t rem0 = (uint32_t)(base - row0 * cpr.d);
    MxRaw8<T> v[U], w[SIGNS ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t l = threadIdx.x + u * 256, n = rem0 + l, r = mx_quot(n, cpr);
        const int c0 = (int)(n - r * cpr.d) * 8;
        const int64_t at = (row0 + r) * C + c0;
        v[u].template load<FULL>(x, at, C - c0, base + l < chunks, C);
        if (SIGNS) w[u].template load<FULL>(sg, at, C - c0, base + l < chunks, C);
    }
    MX_LOADS_OUT();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = base + threadIdx.x + u * 256;
        if (i >= chunks) return;                                         // (chunks is a multiple of 4: a quad stays whole)
        v[u].template fix<FULL>();
        const uint32_t b = mx_scale_byte<FMT>(quad_max_u(v[u].absmax()));
        if (FMT == CN_MX_E2M1) {
            reinterpret_cast<uint32_t*>(codes)[i] = v[u].codes_e2m1(b);
        } else {
            float f[8];
            v[u].get(f);
            reinterpret_cast<uint2*>(codes)[i] = mx_codes_e4m3(f, b);
        }
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)b;
        if (SIGNS) {
            float s[8];
            w[u].template fix<FULL>();
            w[u].get(s);
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m |= (s[j] > 0.f ? 1u : 0u) << j;
            signs[i] = (uint8_t)m;
        }
    }
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            T* __restrict__ out, int64_t chunks, int C, MxDiv cpr, int per) {
    const int64_t base = (int64_t)blockIdx.x * (256 * per);
    const int64_t row0 = base / cpr.d;
    const uint32_t rem0 = (uint32_t)(base - row0 * cpr.d);
    for (int u = 0; u < per; ++u) {
        const uint32_t l = threadIdx.x + u * 256;
        const int64_t i = base + l;
        if (i >= chunks) return;
        const uint32_t n = rem0 + l, r = mx_quot(n, cpr);
        const int c0 = (int)(n - r * cpr.d) * 8;
        const float s = mx_scale_value(scales[i >> 2]);
        float v[8];
        if (FMT == CN_MX_E2M1) {
            mx_values_e2m1(reinterpret_cast<const uint32_t*>(codes)[i], s, v);
        } else {
            const uint2 c = reinterpret_cast<const uint2*>(codes)[i];
            mx_values_e4m3(c.x, c.y, s, v);
        }
        mx_store8(out + (row0 + r) * C + c0, C - c0, v);
    }
}

static int mx_check(const char* who, int64_t rows, int C, int fmt, int dtype) {
    CN_CHECK_ARG(rows >= 0 && C >= 1 && C <= MX_MAX_C, "%s: rows %lld, channels %d (1 .. %d)", who, (long long)rows, C, MX_MAX_C);
    CN_CHECK_ARG(fmt == CN_MX_E2M1 || fmt == CN_MX_E4M3, "%s: unknown format %d", who, fmt);
    CN_CHECK_ARG(dtype == CN_F32 || dtype == CN_BF16, "%s: bad dtype %d", who, dtype);
    CN_CHECK_ARG(rows <= ((int64_t)1 << 40) / C, "%s: tensor too large", who);
    return CN_OK;
}

extern "C" int cn_mx_quantize(const void* x, void* codes, void* scales, const void* sign_src, void* signs, int64_t rows, int C, int fmt,
                              int dtype, void* stream) {
    const int rc = mx_check("cn_mx_quantize", rows, C, fmt, dtype);
    if (rc) return rc;
    CN_CHECK_ARG((sign_src != nullptr) == (signs != nullptr), "cn_mx_quantize: sign_src and signs come together");
    if (rows == 0) return CN_OK;
    CN_CHECK_ARG(x && codes && scales, "cn_mx_quantize: null pointer");
    CN_CHECK_ARG(((uintptr_t)codes & 15) == 0, "cn_mx_quantize: codes must be 16-byte aligned");
    const uint32_t cpr = (uint32_t)cdiv(C, MX_BLOCK) * 4;
    const int64_t chunks = rows * cpr;
    // four chunks a thread (64 or 128 bytes in flight) once that still leaves four workgroups a compute unit.  us, one | four: 16384x256 4.7 |
    // 5.0, 65536x256 11.3 | 10.5, 262144x256 39.5 | 38.1
    const bool many = chunks >= (int64_t)256 * 4 * 1024, full = C % 8 == 0;
    const int64_t grid = (chunks + 256 * (many ? 4 : 1) - 1) / (256 * (many ? 4 : 1));
    CN_CHECK_ARG(mx_grid_fits(grid, 256), "cn_mx_quantize: too many rows for one launch");
#define MX_Q(FMT, SIGNS, U, FULL)                                                                                                      \
    mx_quantize_kernel<T, FMT, SIGNS, U, FULL><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>((const T*)x, (const T*)sign_src,       \
        (uint8_t*)codes, (uint8_t*)scales, (uint8_t*)signs, chunks, C, mx_div(cpr))
#define MX_QU(FMT, SIGNS) do { if (many) { if (full) MX_Q(FMT, SIGNS, 4, true); else MX_Q(FMT, SIGNS, 4, false); } else { if (full) MX_Q(FMT, SIGNS, 1, true); else MX_Q(FMT, SIGNS, 1, false); } } while (0)
    CN_DISPATCH_DTYPE(dtype, T, {
        if (fmt == CN_MX_E2M1) { if (signs) MX_QU(CN_MX_E2M1, true); else MX_QU(CN_MX_E2M1, false); }
        else { if (signs) MX_QU(CN_MX_E4M3, true); else MX_QU(CN_MX_E4M3, false); }
    });
#undef MX_QU
#undef MX_Q
    CN_LAUNCH_CHECK("cn_mx_quantize");
    return CN_OK;
}

extern "C" int cn_mx_dequantize(const void* codes, const void* scales, void* out, int64_t rows, int C, int fmt, int dtype, void* stream) {
    const int rc = mx_check("cn_mx_dequantize", rows, C, fmt, dtype);
    if (rc) return rc;
    if (rows == 0) return CN_OK;
    CN_CHECK_ARG(out && codes && scales, "cn_mx_dequantize: null pointer");
    CN_CHECK_ARG(((uintptr_t)codes & 15) == 0, "cn_mx_dequantize: codes must be 16-byte aligned");
    const uint32_t cpr = (uint32_t)cdiv(C, MX_BLOCK) * 4;
    const int64_t chunks = rows * cpr;
    const int per = chunks >= (int64_t)256 * 4 * 1024 ? 4 : 1;      // us, one | four: 4096x256 4.1 | 4.5, 262144x256 33.6 | 32.0
    const int64_t grid = (chunks + 256 * per - 1) / (256 * per);
    CN_CHECK_ARG(mx_grid_fits(grid, 256), "cn_mx_dequantize: too many rows for one launch");
    CN_DISPATCH_DTYPE(dtype, T, {
        if (fmt == CN_MX_E2M1)
            mx_dequantize_kernel<T, CN_MX_E2M1><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>((const uint8_t*)codes, (const uint8_t*)scales, (T*)out, chunks, C, mx_div(cpr), per);
        else
            mx_dequantize_kernel<T, CN_MX_E4M3><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>((const uint8_t*)codes, (const uint8_t*)scales, (T*)out, chunks, C, mx_div(cpr), per);
    });
    CN_LAUNCH_CHECK("cn_mx_dequantize");
    return CN_OK;
}
