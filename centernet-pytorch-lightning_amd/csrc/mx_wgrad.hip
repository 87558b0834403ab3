// Weight (and bias) gradient of a linear layer / 1x1 convolution from an 8-bit checkpoint of its input:
//   dw[n][k] = sum_r dy[r][n] * x8[r][k],   db[n] = sum_r dy[r][n]
//
// The sum runs over rows, the slow axis of both operands.  Tiles are staged in their natural [row][channel] order — the e4m3 codes
// become bf16 on the way (exact: four significant bits times a power of two; what is below 2^-126 becomes zero) — and the transposing LDS read hands every lane eight
// rows of its channel (rows padded by 64 B: the four rows of a read hit disjoint banks).  A 32-bit dy is split into three bf16 terms
// (8 + 8 + 8 significant bits: nothing is lost from 2^-110 up; below, what lies under bf16's last 2^-133) that share the x8 fragment.
// Row ranges are split over workgroups; their partial sums go to the workspace and are added in a fixed order.  (A join by the workgroup that
// arrives last would save its launch, but its counters would have to live beyond the call, and two captured graphs would share them.)
// Measured: 262144x256x128 bf16 34 us + 6.5 us for the join (136 MB in: 4.0 TB/s; both column tiles ask for dy, memory gives it once),
// 16384x512x2048 55 us = 0.62 PFLOP/s; 1024x2048x512 13 us, 16 row tiles in one workgroup a compute unit: latency.  32 bits: three products,
// 0.42 - 0.7 PFLOP/s (65536x1024x256 142 us).  The large sizes are bound by neither side of the loop alone: matrix pipes are busy 0.24 of
// the time and LDS 0.30 (32 bits: 0.29 and 0.29); a tile's stages — loads' arrival, conversion, two barriers, reads, products — follow
// one another, and two workgroups a compute unit cover that in part.
#include "mx_common.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(8))) short s16x8_t;

// 32(channel) x 16(row) operand out of a [row][channel] LDS tile: lane l gets channel r0 + (l & 31), rows k0 + 8 * (l >> 5) .. + 7
__device__ static inline bf16x8_t mx_tr_frag(const bf16_t* tile, int pitch, int r0, int k0, int lane) {
    const int r = lane & 15, g = lane >> 4;
    const bf16_t* p = tile + (k0 + 8 * (g >> 1) + (r >> 2)) * pitch + r0 + 16 * (g & 1) + 4 * (r & 3);
    typedef __attribute__((address_space(3))) s16x4_t* lds_ptr;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * pitch));
    const s16x8_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8_t, v);
}

struct MxWgGeom {
    const void* dy;
    const uint8_t* codes;
    const uint8_t* scales;
    float* dw;                 // [splits][N][K] partial sums, or the gradient itself (splits == 1)
    float* db;                 // [splits][N], or the gradient itself; nullptr: none
    int64_t rows, per;         // per: rows of one split (a multiple of the row tile)
    int N, K, Kp, blocks;
    int ktiles, accumulate;
};

// a loaded dy chunk into its LDS plane(s)
__device__ static inline void mx_put_dy(const MxRaw8<bf16_t>& r, bf16_t* lds, int) { *reinterpret_cast<u32x4_t*>(lds) = r.a; }
// 32 bits: three planes, `plane` elements apart: truncation to 8 significant bits twice, the rest is exact; an infinity or a NaN is all in
// the first
__device__ static inline void mx_put_dy(const MxRaw8<float>& r, bf16_t* lds, int plane) {
    float f[8];
    r.get(f);
    uint32_t h[8], m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(f[i]);
        const bool fin = (u & 0x7f800000u) != 0x7f800000u;
        h[i] = fin ? u & 0xffff0000u : ((u & 0x7fffffu) ? 0x7fc00000u : u);
        const float d = fin ? f[i] - __uint_as_float(h[i]) : 0.f;
        m[i] = __float_as_uint(d) & 0xffff0000u;
        l[i] = __float_as_uint(d - __uint_as_float(m[i]));
    }
    auto pk = [](const uint32_t (&x)[8]) {
        return u32x4_t{(x[0] >> 16) | (x[1] & 0xffff0000u), (x[2] >> 16) | (x[3] & 0xffff0000u), (x[4] >> 16) | (x[5] & 0xffff0000u), (x[6] >> 16) | (x[7] & 0xffff0000u)};
    };
    *reinterpret_cast<u32x4_t*>(lds) = pk(h);
    *reinterpret_cast<u32x4_t*>(lds + plane) = pk(m);
    *reinterpret_cast<u32x4_t*>(lds + 2 * plane) = pk(l);
}

template <typename R> __device__ static inline void mx_buf8(MxRaw8<bf16_t>& w, R rsrc, uint32_t ofs) {
    w.a = __builtin_amdgcn_raw_buffer_load_b128(rsrc, ofs, 0, 0);
}
template <typename R> __device__ static inline void mx_buf8(MxRaw8<float>& w, R rsrc, uint32_t ofs) {
    w.a = __builtin_amdgcn_raw_buffer_load_b128(rsrc, ofs, 0, 0);
    w.b = __builtin_amdgcn_raw_buffer_load_b128(rsrc, ofs + 16, 0, 0);
}

template <typename T, int TN, int TK, bool FULL>
__global__ __launch_bounds__(256) void mx_wgrad_kernel(const MxWgGeom g) {
    constexpr int NP = sizeof(T) == 2 ? 1 : 3;
    constexpr int BR = 64;                                        // rows per tile
    constexpr int YP = TN + 32, XP = TK + 32;                     // LDS pitches (elements)
    constexpr int YV = BR * TN / 8 / 256, XV = BR * TK / 16 / 256;
    constexpr int YC = TN / 8, XC = TK / 16;
    constexpr int MI = TN / 64, NJ = TK / 64;                     // 2 x 2 waves of 32 x 32 tiles
    // tiles in flight.  In the narrow ones a second pays for 16 bits (quantising and gradient of 1024x2048x512, one | two: 18.8 | 17.4 us), not
    // for 32 (5883x208x80 15.5 | 16.4).  In the wide ones it is not measured: 16 bits take 146 of the 256 registers that their two waves a
    // SIMD have, and a second tile 26 more
    constexpr int DEEP = sizeof(T) == 2 && TN * TK == 64 * 64 ? 2 : 1;
    constexpr int PLANE = BR * YP;
    __shared__ __attribute__((aligned(16))) bf16_t lds[NP * PLANE + BR * XP];
    bf16_t* const ly = lds;
    bf16_t* const lx = lds + NP * PLANE;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    const int nt = blockIdx.y / g.ktiles, kt = blockIdx.y - nt * g.ktiles;
    const int n0 = nt * TN, k0 = kt * TK;
    const int64_t rbeg = (int64_t)blockIdx.x * g.per, rend = rbeg + g.per < g.rows ? rbeg + g.per : g.rows;
    const bool bias = g.db != nullptr && kt == 0;

    const int yc = (tid % YC) * 8, yr = tid / YC;                 // dy: chunk column (the same for all YV loads), first row
    const int xc = (tid % XC) * 16, xr = tid / XC;
    const int yleft = g.N - n0 - yc;
    const bool xok = k0 + xc < g.Kp;                              // (Kp is a multiple of 32: 16 codes are inside or outside)

    // raw tiles on their way, asked for DEEP tiles ahead of their use.  FULL (N a multiple of 8, dy on a 16-byte
    // border): buffer loads whose range ends with the rows — what lies behind reads as zero, and the lanes' offsets are the same for
    // every tile (columns behind the last: an offset out of range; offsets stay below 2^31 + 2^26, and all of one is in the lane's part:
    // the range check subtracts a scalar part from the range, which wraps where that is the larger).
    struct Raw { MxRaw8<T> y[YV]; u32x4_t x[XV]; uint32_t s[XV]; };
    Raw ra, rb;
    constexpr uint32_t OUT = 0x80000000u;
    const uint32_t yofs = yleft > 0 ? (uint32_t)(yr * g.N + n0 + yc) * sizeof(T) : OUT;
    const uint32_t xofs = xok ? (uint32_t)(xr * g.Kp + k0 + xc) : OUT, sofs = xok ? (uint32_t)(xr * g.blocks + ((k0 + xc) >> 5)) : OUT;
    auto gload = [&](Raw& w, int64_t r0) {
        const int left = r0 < rend ? (rend - r0 < BR ? (int)(rend - r0) : BR) : 0;         // rows of this tile
        const int64_t rr = left ? r0 : rbeg;
        if (FULL) {
            const auto by = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(reinterpret_cast<const T*>(g.dy) + rr * g.N), 0, (uint32_t)left * g.N * sizeof(T), 0x00020000);
#pragma unroll
            for (int v = 0; v < YV; ++v) mx_buf8(w.y[v], by, yofs + (uint32_t)(v * (256 / YC)) * g.N * sizeof(T));
        } else {
#pragma unroll
            for (int v = 0; v < YV; ++v) {
                const int r = yr + v * (256 / YC);
                w.y[v].template load<false>(reinterpret_cast<const T*>(g.dy), (rr + r) * g.N + n0 + yc, yleft, r < left, g.N);
            }
        }
        const auto bx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.codes + rr * g.Kp), 0, (uint32_t)left * g.Kp, 0x00020000);
        const auto bs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.scales + rr * g.blocks), 0, (uint32_t)left * g.blocks, 0x00020000);
#pragma unroll
        for (int v = 0; v < XV; ++v) {
            w.x[v] = __builtin_amdgcn_raw_buffer_load_b128(bx, xofs + (uint32_t)(v * (256 / XC)) * g.Kp, 0, 0);
            w.s[v] = __builtin_amdgcn_raw_buffer_load_b8(bs, sofs + (uint32_t)(v * (256 / XC)) * g.blocks, 0, 0);
        }
    };
    float sb[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sb[j] = 0.f;
    auto lstore = [&](Raw& w) {
#pragma unroll
        for (int v = 0; v < YV; ++v) {
            if (!FULL) w.y[v].template fix<false>();              // (ranged buffer loads leave nothing to put right)
            mx_put_dy(w.y[v], ly + (yr + v * (256 / YC)) * YP + yc, PLANE);
            if (bias) {
                float f[8];
                w.y[v].get(f);
#pragma unroll
                for (int j = 0; j < 8; ++j) sb[j] += f[j];
            }
        }
#pragma unroll
        for (int v = 0; v < XV; ++v) {
            const float s = mx_scale_value(w.s[v]);
            const uint32_t q[4] = {w.x[v].x, w.x[v].y, w.x[v].z, w.x[v].w};
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], s, false));
                o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], s, true));
            }
            bf16_t* p = lx + (xr + v * (256 / XC)) * XP + xc;
            st16(p, make_uint4(o[0], o[1], o[2], o[3]));
            st16(p + 8, make_uint4(o[4], o[5], o[6], o[7]));
        }
    };

    f32x16_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    auto tile = [&](Raw& w, int64_t r0) {
        __syncthreads();                                          // the previous tile has been read
        lstore(w);
        __syncthreads();
        gload(w, r0 + DEEP * BR);                                 // (behind the end: zeros)
#pragma unroll
        for (int s = 0; s < BR / 16; ++s) {
            bf16x8_t b[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) b[j] = mx_tr_frag(lx, XP, (wn * NJ + j) * 32, s * 16, lane);
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const bf16x8_t a = mx_tr_frag(ly + p * PLANE, YP, (wm * MI + i) * 32, s * 16, lane);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
                }
        }
    };
    gload(ra, rbeg);
    if (DEEP == 1) {
        for (int64_t r0 = rbeg; r0 < rend; r0 += BR) tile(ra, r0);
    } else {
        gload(rb, rbeg + BR);
        for (int64_t r0 = rbeg; r0 < rend; r0 += 2 * BR) {
            tile(ra, r0);
            if (r0 + BR < rend) tile(rb, r0 + BR);
        }
    }

    float* dw = g.dw + (int64_t)blockIdx.x * g.N * g.K;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int k = k0 + (wn * NJ + j) * 32 + (lane & 31);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = n0 + (wm * MI + i) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                if (n < g.N && k < g.K) {
                    float* p = dw + (int64_t)n * g.K + k;
                    *p = g.accumulate ? *p + acc[i][j][e] : acc[i][j][e];
                }
            }
        }
    if (bias) {
        float* red = reinterpret_cast<float*>(lds);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) red[tid * 8 + j] = sb[j];
        __syncthreads();
        if (tid < TN) {
            float s = 0.f;
            for (int q = 0; q < 256 / YC; ++q) s += red[(q * YC + (tid >> 3)) * 8 + (tid & 7)];
            float* p = g.db + (int64_t)blockIdx.x * g.N + n0 + tid;
            if (n0 + tid < g.N) *p = g.accumulate ? *p + s : s;
        }
    }
}

// out[i] = (accumulate ? out[i] : 0) + sum_s part[s][i] for i < n (dw) and then n <= i < n + nb (db).  GS split groups of 256 / GS threads,
// four outputs a thread; the groups meet in LDS in order.
template <int GS>
__global__ __launch_bounds__(256) void mx_wgrad_join_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n, int splits,
                                                            const float* __restrict__ part_b, float* __restrict__ out_b, int nb, int accumulate) {
    constexpr int TO = 256 / GS;
    __shared__ float red[GS][TO * 4];
    const int o = threadIdx.x % TO, gs = threadIdx.x / TO;
    const int64_t wgs_w = (n + TO * 4 - 1) / (TO * 4);             // workgroups of dw come first
    const bool w = blockIdx.x < wgs_w;
    const int64_t len = w ? n : nb, i0 = ((int64_t)blockIdx.x - (w ? 0 : wgs_w)) * (TO * 4) + o * 4;
    const float* p = (w ? part : part_b) + i0;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i0 + 4 <= len) {
#pragma unroll 8
        for (int k = gs; k < splits; k += GS) {
            const u32x4_t v = *reinterpret_cast<const u32x4_a4*>(p + k * len);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += __uint_as_float(v[j]);
        }
    } else {
        for (int k = gs; k < splits; k += GS)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += i0 + j < len ? p[k * len + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[gs][o * 4 + j] = s[j];
    __syncthreads();
    for (int t = threadIdx.x; t < TO * 4; t += 256) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < GS; ++k) v += red[k][t];
        const int64_t i = i0 - o * 4 + t;
        if (i < len) {
            float* q = (w ? out : out_b) + i;
            *q = accumulate ? *q + v : v;
        }
    }
}

// Tiles and splits.  Large problems take the wide tiles (a row of dy / x8 is read again for every K / N tile) and two workgroups a compute
// unit; small ones the narrow tiles, whose workgroups are short of work sooner.  A split writes and reads a whole dw and the join is a
// launch of its own: none once the tiles alone fill the card, or for a few rows of many tiles, and two row tiles to a split at least.
// us, wide | narrow, bf16: 262144x256x128 43 | 56, 65536x1024x256 53 | 72, 16384x512x2048 56 | 74, 25394x224x660 31 | 46;
// 8192x512x512 24.3 | 21.8, 65536x256x64 18.5 | 15.2, 4096x1024x256 19.1 | 16.5, 1024x2048x512 18.3 | 12.4 (15.8 in two splits),
// 204x800x732 7.4 (10.6 in two splits), 15993x22x51 10.9 (13.2 with a row tile a split).
// The border goes by products alone.  Below it, gradient alone, wide | narrow: 131072x128x128 22.8 | 19.7, 65536x256x128 21.1 | 18.8, 16384x256x512
// 20.1 | 19.2, 2048x1024x1024 26.5 | 21.0; only many rows of one tile would be better off wide: 262144x128x80 23.7 | 26.7, 262144x80x80 21.9 | 25.9.
// 32 bits (64 x 128 | 64 x 64): 65536x1024x256 137 | 176, 65536x256x64 20.4 | 22.7, 30000x80x208 20.2 | 24.0; 831x864x560 17.1 | 16.2.
struct MxWgPlan { bool wide; int tn, tk, ntiles, ktiles, splits; int64_t per; };
static MxWgPlan mxwg_plan(int64_t rows, int K, int N, int dtype) {
    MxWgPlan p;
    const double macs = (double)rows * K * N;
    p.wide = dtype == CN_BF16 ? (macs >= 3e9 && N > 64 && K > 64) : (macs >= 5e8 && K > 64);
    p.tn = p.wide && dtype == CN_BF16 ? 128 : 64;
    p.tk = p.wide ? 128 : 64;
    p.ntiles = cdiv(N, p.tn);
    p.ktiles = cdiv(K, p.tk);
    const int64_t tiles = (int64_t)p.ntiles * p.ktiles, rtiles = (rows + 63) / 64;
    int64_t s = tiles >= 192 || (rtiles <= 16 && tiles >= 32) ? 1 : 512 / tiles;
    s = s < rtiles / 2 ? s : rtiles / 2;
    s = s < 1 ? 1 : s;
    p.per = (rtiles + s - 1) / s * 64;
    p.splits = (int)((rows + p.per - 1) / p.per);
    return p;
}

extern "C" size_t cn_mx_linear_wgrad_bytes(int64_t rows, int K, int N, int dtype) {
    if (rows < 1 || K < 1 || N < 1 || K > MX_MAX_C || N > MX_MAX_C) return 0;
    const MxWgPlan p = mxwg_plan(rows, K, N, dtype);
    return p.splits > 1 ? sizeof(float) * (size_t)p.splits * ((size_t)N * K + N) : 0;
}

extern "C" int cn_mx_linear_wgrad_variant(int64_t rows, int K, int N, int dtype) {
    if (rows < 1 || K < 1 || N < 1 || K > MX_MAX_C || N > MX_MAX_C) return 0;
    const MxWgPlan p = mxwg_plan(rows, K, N, dtype);
    return p.tn * 1000000 + p.tk * 1000 + p.splits;
}

template <typename T, int TN, int TK>
static void mxwg_launch(const MxWgGeom& g, const MxWgPlan& p, hipStream_t st) {
    const dim3 grid(p.splits, p.ntiles * p.ktiles);
    if (g.N % 8 == 0 && ((uintptr_t)g.dy & 15) == 0) mx_wgrad_kernel<T, TN, TK, true><<<grid, 256, 0, st>>>(g);
    else mx_wgrad_kernel<T, TN, TK, false><<<grid, 256, 0, st>>>(g);
}

extern "C" int cn_mx_linear_wgrad(const void* dy, const void* codes, const void* scales, float* dw, float* db, int accumulate, int64_t rows,
                                  int K, int N, int dtype, void* ws, size_t ws_bytes, void* stream) {
    CN_CHECK_ARG(rows >= 1 && K >= 1 && N >= 1 && K <= MX_MAX_C && N <= MX_MAX_C && rows <= ((int64_t)1 << 40) / (K > N ? K : N),
                 "cn_mx_linear_wgrad: rows %lld, K %d, N %d", (long long)rows, K, N);
    CN_CHECK_ARG(dtype == CN_F32 || dtype == CN_BF16, "cn_mx_linear_wgrad: bad dtype %d", dtype);
    CN_CHECK_ARG(dy && codes && scales && dw, "cn_mx_linear_wgrad: null pointer");
    CN_CHECK_ARG(((uintptr_t)codes & 15) == 0, "cn_mx_linear_wgrad: codes must be 16-byte aligned");
    if (ws_bytes < cn_mx_linear_wgrad_bytes(rows, K, N, dtype) || (!ws && ws_bytes)) {
        cn_set_error("cn_mx_linear_wgrad: workspace of %zu bytes needed", cn_mx_linear_wgrad_bytes(rows, K, N, dtype));
        return CN_EWORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    const MxWgPlan p = mxwg_plan(rows, K, N, dtype);
    CN_CHECK_ARG((int64_t)p.ntiles * p.ktiles <= 65535, "cn_mx_linear_wgrad: K x N too large");
    const bool join = p.splits > 1;
    MxWgGeom g;
    g.dy = dy;
    g.codes = (const uint8_t*)codes;
    g.scales = (const uint8_t*)scales;
    g.dw = join ? (float*)ws : dw;
    g.db = db ? (join ? (float*)ws + (size_t)p.splits * N * K : db) : nullptr;
    g.rows = rows;
    g.per = p.per;
    g.N = N;
    g.K = K;
    g.blocks = cdiv(K, MX_BLOCK);
    g.Kp = g.blocks * MX_BLOCK;
    g.ktiles = p.ktiles;
    g.accumulate = join ? 0 : accumulate;
    if (dtype == CN_BF16) {
        if (p.wide) mxwg_launch<bf16_t, 128, 128>(g, p, st);
        else mxwg_launch<bf16_t, 64, 64>(g, p, st);
    } else {
        if (p.wide) mxwg_launch<float, 64, 128>(g, p, st);
        else mxwg_launch<float, 64, 64>(g, p, st);
    }
    CN_LAUNCH_CHECK("cn_mx_linear_wgrad");
    if (join) {
        const int64_t n = (int64_t)N * K;
        const int nb = db ? N : 0;
        // more groups where the splits are many and the outputs few; 16 / 64 / 1024 outputs a workgroup.  us, 64 | 16 | 1 groups: 15993x22x51
        // 8.8 | 10.9 | 28, 65536x64x64 16.1 | 13.6 | 34, 65536x256x64 18.1 | 15.3 | 19.9; 8192x512x512 (few splits) 29.8 | 22.4 | 22.2
        if (p.splits >= 64 && n <= 2048) mx_wgrad_join_kernel<64><<<(unsigned)(cdiv(n, 16) + cdiv(nb, 16)), 256, 0, st>>>(g.dw, dw, n, p.splits, g.db, db, nb, accumulate);
        else if (p.splits >= 16) mx_wgrad_join_kernel<16><<<(unsigned)(cdiv(n, 64) + cdiv(nb, 64)), 256, 0, st>>>(g.dw, dw, n, p.splits, g.db, db, nb, accumulate);
        else mx_wgrad_join_kernel<1><<<(unsigned)(cdiv(n, 1024) + cdiv(nb, 1024)), 256, 0, st>>>(g.dw, dw, n, p.splits, g.db, db, nb, accumulate);
        CN_LAUNCH_CHECK("cn_mx_linear_wgrad");
    }
    return CN_OK;
}
