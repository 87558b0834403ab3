// y = act(x4 @ w4^T + bias + residual): x [M][K] is quantised to e2m1 on the way in (one scale per 32 channels, mx_common.h), w [N][K]
// was quantised and laid out once (cn_mx_pack_weight).  Products of 4-bit values times powers of two are exact, sums are fp32
// (v_mfma_scale_f32_32x32x64_f8f6f4: a lane's 16 bytes are one block of 32 channels, its scale rides in a byte of a register).
//
// What has to move is x in and y out; the codes of x never leave the workgroup.  A workgroup quantises its BM rows once into LDS and
// keeps them there while it walks all its columns, so x is read from memory once whatever N is; the weights stream from L2 in
// fragment order (1 KB contiguous per 32 columns x 64 channels).  K beyond what LDS holds is taken in chunks.
#include "mx_common.h"

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

// ---- weights: codes [ceil(N/32)][S][64 lanes][16 B], then scales [ceil(N/32)][ceil(S/4)][64 lanes][4 B], S = ceil(K/64) ------------
// lane l: column l & 31 of the tile, block 2 s + (l >> 5); byte s & 3 of the scale word belongs to step s.  Filler: codes 0, scale 1.
static inline int64_t mxw_codes_bytes(int N, int K) { return (int64_t)cdiv(N, 32) * cdiv(K, 64) * 1024; }

template <typename T>
__global__ __launch_bounds__(64) void mx_pack_weight_kernel(const T* __restrict__ w, uint4* __restrict__ codes, uint32_t* __restrict__ scales,
                                                            int N, int K, int S) {
    const int lane = threadIdx.x, nt = blockIdx.y, t = blockIdx.x, n = nt * 32 + (lane & 31);
    uint32_t sw = 0;
    for (int i = 0; i < 4; ++i) {
        const int s = 4 * t + i, k0 = (2 * s + (lane >> 5)) * 32;
        uint32_t b = 127;
        if (s < S) {
            float v[4][8];
            uint32_t m = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                mx_load8(w + (int64_t)n * K + k0 + q * 8, n < N ? K - k0 - q * 8 : 0, v[q]);
                const uint32_t a = mx_absmax8(v[q]);
                m = a > m ? a : m;
            }
            b = mx_scale_byte<CN_MX_E2M1>(m);
            codes[((int64_t)nt * S + s) * 64 + lane] = make_uint4(mx_codes_e2m1(v[0], b), mx_codes_e2m1(v[1], b), mx_codes_e2m1(v[2], b), mx_codes_e2m1(v[3], b));
        }
        sw |= b << (8 * i);
    }
    scales[((int64_t)nt * gridDim.x + t) * 64 + lane] = sw;
}

extern "C" size_t cn_mx_weight_bytes(int N, int K) {
    if (N < 1 || K < 1 || N > MX_MAX_C || K > MX_MAX_C) return 0;
    return (size_t)mxw_codes_bytes(N, K) + (size_t)cdiv(N, 32) * cdiv(cdiv(K, 64), 4) * 256;
}

extern "C" int cn_mx_pack_weight(const void* w, void* packed, int N, int K, int dtype, void* stream) {
    CN_CHECK_ARG(N >= 1 && K >= 1 && N <= MX_MAX_C && K <= MX_MAX_C, "cn_mx_pack_weight: N %d, K %d (1 .. %d)", N, K, MX_MAX_C);
    CN_CHECK_ARG(dtype == CN_F32 || dtype == CN_BF16, "cn_mx_pack_weight: bad dtype %d", dtype);
    CN_CHECK_ARG(w && packed && ((uintptr_t)packed & 15) == 0, "cn_mx_pack_weight: null or misaligned pointer");
    const int S = cdiv(K, 64);
    uint32_t* scales = (uint32_t*)((char*)packed + mxw_codes_bytes(N, K));
    CN_DISPATCH_DTYPE(dtype, T, {
        mx_pack_weight_kernel<T><<<dim3(cdiv(S, 4), cdiv(N, 32)), 64, 0, (hipStream_t)stream>>>((const T*)w, (uint4*)packed, scales, N, K, S);
    });
    CN_LAUNCH_CHECK("cn_mx_pack_weight");
    return CN_OK;
}

// ---- product -----------------------------------------------------------------------------------------------------------------------
struct MxLinGeom {
    const void* x;
    const uint4* wc;
    const uint32_t* ws;
    const float* bias;
    const void* res;
    void* y;
    int64_t M;
    int K, N, S, S4;           // S: steps of 64 channels, S4 = ceil(S / 4)
    int chunk;                 // steps that LDS holds (a multiple of 4 unless it is S)
    int ntiles;                // 64-column tiles in all
    int per_wg;                // passes over the waves' columns per workgroup
    int relu;
    int pitch, spitch;         // LDS bytes per row: codes, scales
    MxDiv cdiv_full, cdiv_last;        // 8-channel pieces per row of a full / the last chunk
    int sc_ofs, ep_ofs;        // LDS offsets of the scales and of the output staging
};

#define MXL_EP 68              // floats per staged output row (64 + 4: rows on different banks)

template <typename T, int BM, int WM>
__global__ __launch_bounds__(256) void mx_linear_kernel(const MxLinGeom g) {
    constexpr int WN = 4 / WM, MI = BM / WM / 32;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    const int64_t m0 = (int64_t)blockIdx.x * BM;
    const int rows = (int)(g.M - m0 < BM ? g.M - m0 : BM);
    const T* __restrict__ X = reinterpret_cast<const T*>(g.x) + m0 * g.K;

    auto stage = [&](int s0, int s1) {                            // quantise channels 64 s0 .. 64 s1 of the workgroup's rows into LDS
        const MxDiv dv = s1 == g.S ? g.cdiv_last : g.cdiv_full;
        const int total = BM * (int)dv.d;
        constexpr int U = 4;
        for (int base = tid; base < total; base += 256 * U) {
            float v[U][8];
            int row[U], pc[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = base + u * 256;
                row[u] = (int)mx_quot(i, dv);
                pc[u] = (int)i - row[u] * (int)dv.d;
                const int c0 = s0 * 64 + pc[u] * 8;
                mx_load8(X + (int64_t)row[u] * g.K + c0, ((int)i < total && row[u] < rows) ? g.K - c0 : 0, v[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t b = mx_scale_byte<CN_MX_E2M1>(quad_max_u(mx_absmax8(v[u])));
                if (base + u * 256 < total) {                     // (whole quads)
                    *reinterpret_cast<uint32_t*>(smem + row[u] * g.pitch + pc[u] * 4) = mx_codes_e2m1(v[u], b);
                    const int blk = pc[u] >> 2, s = blk >> 1;     // byte s & 3 of word (s / 4, half)
                    if ((pc[u] & 3) == 0) smem[g.sc_ofs + row[u] * g.spitch + ((s >> 2) * 2 + (blk & 1)) * 4 + (s & 3)] = (uint8_t)b;
                }
            }
        }
    };

    const bool resident = g.chunk >= g.S;
    if (resident) { stage(0, g.S); __syncthreads(); }

    const unsigned char* arow = smem + (wm * MI * 32 + (lane & 31)) * g.pitch + (lane >> 5) * 16;
    const unsigned char* srow = smem + g.sc_ofs + (wm * MI * 32 + (lane & 31)) * g.spitch + (lane >> 5) * 4;
    float* ep = reinterpret_cast<float*>(smem + g.ep_ofs) + wave * 32 * MXL_EP;

    for (int it = 0; it < g.per_wg; ++it) {
        const int tile = (blockIdx.y * g.per_wg + it) * WN + wn;  // 64 columns
        const bool live = tile < g.ntiles;
        if (resident && !live) break;                             // (no barrier below in the resident form)
        const int t32 = (g.N + 31) >> 5, nt0 = live ? tile * 2 : 0, nt1 = nt0 + 1 < t32 ? nt0 + 1 : nt0;   // (an odd count: the last tile twice)
        f32x16_t acc[MI][2];
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

        for (int s0 = 0; s0 < g.S; s0 += g.chunk) {
            const int s1 = s0 + g.chunk < g.S ? s0 + g.chunk : g.S;
            if (!resident) {
                __syncthreads();
                stage(s0, s1);
                __syncthreads();
            }
            const uint4* b0 = g.wc + (int64_t)nt0 * g.S * 64 + lane;
            const uint4* b1 = g.wc + (int64_t)nt1 * g.S * 64 + lane;
            const uint32_t* q0 = g.ws + (int64_t)nt0 * g.S4 * 64 + lane;
            const uint32_t* q1 = g.ws + (int64_t)nt1 * g.S4 * 64 + lane;
            for (int t = s0 >> 2; 4 * t < s1; ++t) {
                const uint32_t sb0 = q0[t * 64], sb1 = q1[t * 64];
                uint32_t sa[MI];
#pragma unroll
                for (int i = 0; i < MI; ++i) sa[i] = *reinterpret_cast<const uint32_t*>(srow + i * 32 * g.spitch + (t - (s0 >> 2)) * 8);
                uint4 fb[4][2];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int s = 4 * t + u < s1 ? 4 * t + u : s1 - 1;
                    fb[u][0] = ldg16(b0 + s * 64);
                    fb[u][1] = ldg16(b1 + s * 64);
                }
#define MXL_STEP(u)                                                                                                                     \
    if (4 * t + u < s1) {                                                                                                               \
        _Pragma("unroll") for (int i = 0; i < MI; ++i) {                                                                                \
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(arow + i * 32 * g.pitch + (4 * t + u - s0) * 32);                       \
            const i32x8_t av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};                                                    \
            _Pragma("unroll") for (int j = 0; j < 2; ++j) {                                                                             \
                const i32x8_t bv = {(int)fb[u][j].x, (int)fb[u][j].y, (int)fb[u][j].z, (int)fb[u][j].w, 0, 0, 0, 0};                    \
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc[i][j], 4, 4, u, (int)sa[i], u, (int)(j ? sb1 : sb0)); \
            }                                                                                                                           \
        }                                                                                                                               \
    }
                MXL_STEP(0) MXL_STEP(1) MXL_STEP(2) MXL_STEP(3)
#undef MXL_STEP
            }
        }
        if (!live) continue;

        // 32 rows at a time through LDS (a wave's own slice: no barrier), then 8 columns a lane
        const int n0 = tile * 64, nc = n0 + (lane & 7) * 8, left = g.N - nc;
        float bs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) bs[e] = (g.bias && e < left) ? g.bias[nc + e] : 0.f;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) ep[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * MXL_EP + j * 32 + (lane & 31)] = acc[i][j][e];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = q * 8 + (lane >> 3);
                const int64_t m = m0 + (wm * MI + i) * 32 + r;
                float v[8];
                const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(ep + r * MXL_EP + (lane & 7) * 8);
                const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(ep + r * MXL_EP + (lane & 7) * 8 + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = lo[e] + bs[e]; v[4 + e] = hi[e] + bs[4 + e]; }
                if (m < g.M && left > 0) {
                    if (g.res) {
                        float rv[8];
                        mx_load8(reinterpret_cast<const T*>(g.res) + m * g.N + nc, left, rv);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += rv[e];
                    }
                    if (g.relu) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];        // (a NaN stays one)
                    }
                    mx_store8(reinterpret_cast<T*>(g.y) + m * g.N + nc, left, v);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

template <typename T, int BM, int WM>
static int mxl_launch(MxLinGeom g, hipStream_t st) {
    constexpr int WN = 4 / WM;
    // LDS: at most 1024 steps' worth is never needed; hold as many channels as fit beside the output staging
    const int ep = 4 * 32 * MXL_EP * 4;
    int chunk = g.S;
    auto bytes = [&](int c, int* pitch, int* spitch) {
        *pitch = c * 32 + 16;                       // an odd number of 16-byte pieces: eight rows' reads hit different banks
        *spitch = cdiv(c, 4) * 8 + 4;
        return BM * (*pitch + *spitch);
    };
    while (bytes(chunk, &g.pitch, &g.spitch) + ep > 150 * 1024) chunk = chunk > 64 ? 64 : chunk / 2 / 4 * 4;
    g.chunk = chunk;
    g.sc_ofs = BM * g.pitch;
    g.ep_ofs = (BM * (g.pitch + g.spitch) + 15) / 16 * 16;
    const int smem = g.ep_ofs + ep;
    g.cdiv_full = mx_div((uint32_t)chunk * 8);
    const int last = g.S % chunk ? g.S % chunk : chunk;
    g.cdiv_last = mx_div((uint32_t)last * 8);
    g.ntiles = cdiv(g.N, 64);
    const int64_t mt = (g.M + BM - 1) / BM;
    if (mt >= ((int64_t)1 << 31)) { cn_set_error("cn_mx_linear_fwd: too many rows"); return CN_EINVAL; }
    const int passes = cdiv(g.ntiles, WN);
    // one workgroup walks all columns of its rows unless that leaves compute units idle
    int split = (int)(mt >= 512 ? 1 : (512 + mt - 1) / mt);
    split = chunk < g.S ? passes : (split < passes ? split : passes);
    g.per_wg = cdiv(passes, split);
    split = cdiv(passes, g.per_wg);
    static bool attr[64] = {};
    int dev = 0;
    (void)hipGetDevice(&dev);
    dev &= 63;
    if (!attr[dev]) {
        CN_HIP(hipFuncSetAttribute((const void*)mx_linear_kernel<T, BM, WM>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        attr[dev] = true;
    }
    mx_linear_kernel<T, BM, WM><<<dim3((unsigned)mt, split), 256, smem, st>>>(g);
    CN_LAUNCH_CHECK("cn_mx_linear_fwd");
    return CN_OK;
}

extern "C" int cn_mx_linear_fwd(const void* x, const void* packed, const float* bias, const void* residual, void* y, int64_t M, int K, int N,
                                int relu, int dtype, void* stream) {
    CN_CHECK_ARG(M >= 0 && K >= 1 && N >= 1 && K <= MX_MAX_C && N <= MX_MAX_C && M <= ((int64_t)1 << 40) / (K > N ? K : N),
                 "cn_mx_linear_fwd: M %lld, K %d, N %d", (long long)M, K, N);
    CN_CHECK_ARG(dtype == CN_F32 || dtype == CN_BF16, "cn_mx_linear_fwd: bad dtype %d", dtype);
    if (M == 0) return CN_OK;
    CN_CHECK_ARG(x && packed && y && ((uintptr_t)packed & 15) == 0, "cn_mx_linear_fwd: null or misaligned pointer");
    MxLinGeom g;
    memset(&g, 0, sizeof(g));
    g.x = x;
    g.wc = (const uint4*)packed;
    g.ws = (const uint32_t*)((const char*)packed + mxw_codes_bytes(N, K));
    g.bias = bias;
    g.res = residual;
    g.y = y;
    g.M = M;
    g.K = K;
    g.N = N;
    g.S = cdiv(K, 64);
    g.S4 = cdiv(g.S, 4);
    g.relu = relu;
    hipStream_t st = (hipStream_t)stream;
#define MXL_GO(BM, WM) return dtype == CN_BF16 ? mxl_launch<bf16_t, BM, WM>(g, st) : mxl_launch<float, BM, WM>(g, st)
    if (M <= 64) { MXL_GO(32, 1); }
    if (N <= 64) { MXL_GO(128, 4); }
    if (N <= 128) { MXL_GO(128, 2); }
    if (K <= 512) { MXL_GO(128, 1); }
    MXL_GO(64, 1);
#undef MXL_GO
}
