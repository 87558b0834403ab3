// Backward of training-mode BatchNorm (+ ReLU, + residual input) from an 8-bit checkpoint of its input.
//
//   d       = dy where the layer's output was positive (the checkpoint's sign bits), else 0      (no ReLU: d = dy)
//   dbeta_c = sum_r d,   dgamma_c = invstd_c * sum_r d (x8 - mean_c)
//   dx      = gamma invstd (d - dbeta / R - xhat dgamma / R) = a d - b (x8 - mean) - c,   dres = d (+ racc)
//
// x8 is what the e4m3 codes stand for.  The sums need every row before the first dx, so dy and the codes are read twice: 2 x 3.16
// bytes per bf16 element in, 2 (4 with a residual input) out.  A thread owns eight channels and walks rows, so the sums and the
// coefficients stay in registers; partial sums are joined in a fixed order (results do not depend on the schedule).
// Bound by memory: 262144 x 256 bf16, with ReLU, sums 39 us (211 MB, 5.4 TB/s), finish 5, dx 74 (345 MB, 4.7 TB/s: reads and writes mixed);
// 512 x 512 7.1 us in one launch.
#include "mx_common.h"

struct MxBnGeom {
    const void* dy;
    const uint8_t* codes;
    const uint8_t* scales;
    const uint8_t* signs;      // nullptr: no ReLU
    int64_t rows;
    int C, cpr, blocks;        // cpr: 8-channel chunks per (padded) row of codes, blocks = cpr / 4
    int ld;                    // C rounded up to 8: channels per row of the partial sums and of the coefficients
    int lg;                    // log2 of the chunks a workgroup covers
    int64_t per;               // rows per workgroup of the apply pass
};

#define MXBN_U 4               // rows a thread has in flight

// a row's dy, codes, scale and sign bits for a thread's chunk, as they lie in memory
template <typename T> struct MxBnRow {
    MxRaw8<T> dy;
    uint2 q;
    uint32_t b, m;
    template <bool SIGNS, bool FULL> __device__ inline void load(const MxBnGeom& g, int64_t r, int c, int left, bool ok) {
        r = ok ? r : 0;                                           // (row 0 is readable; its values are not used then)
        const int64_t i = r * g.cpr + c;
        q = reinterpret_cast<const uint2*>(g.codes)[i];
        b = g.scales[r * g.blocks + (c >> 2)];
        m = SIGNS ? g.signs[i] : 0u;
        dy.template load<FULL>(reinterpret_cast<const T*>(g.dy), r * g.C + c * 8, left, true, g.C);
    }
    template <bool SIGNS, bool FULL> __device__ inline void get(float (&d)[8], float (&v)[8]) {
        dy.template fix<FULL>();
        dy.get(d);
        if (SIGNS) {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = (m >> j) & 1 ? d[j] : 0.f;
        }
        mx_values_e4m3(q.x, q.y, mx_scale_value(b), v);
    }
};

// The workgroups walk the rows side by side (in step with time), and the apply pass starts at the end: what was read last is still in the
// memory-side cache (45 -> 40 us and 76 -> 74 us at 262144 x 256).
template <typename T, bool SIGNS, bool FULL>
__global__ __launch_bounds__(256) void mx_bn_sums_kernel(const MxBnGeom g, const float* __restrict__ mean, float* __restrict__ part) {
    __shared__ float red[4 * 32 * 16];
    const int tid = threadIdx.x, tc = 1 << g.lg, cl = tid & (tc - 1), rl = tid >> g.lg, nrl = 256 >> g.lg;
    const int c = blockIdx.y * tc + cl, left = g.C - c * 8;
    float s0[8], s1[8], mu[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { s0[j] = 0.f; s1[j] = 0.f; mu[j] = j < left ? mean[c * 8 + j] : 0.f; }
    if (left > 0) {
        for (int64_t r = (int64_t)blockIdx.x * (MXBN_U * nrl) + rl; r < g.rows; r += (int64_t)gridDim.x * (MXBN_U * nrl)) {
            MxBnRow<T> row[MXBN_U];
#pragma unroll
            for (int u = 0; u < MXBN_U; ++u) row[u].template load<SIGNS, FULL>(g, r + u * nrl, c, left, r + u * nrl < g.rows);
            MX_LOADS_OUT();
#pragma unroll
            for (int u = 0; u < MXBN_U; ++u) {
                if (r + u * nrl < g.rows) {
                    float d[8], v[8];
                    row[u].template get<SIGNS, FULL>(d, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) { s0[j] += d[j]; s1[j] = fmaf(d[j], v[j] - mu[j], s1[j]); }
                }
            }
        }
    }
    // lanes of one chunk within the wave, then the four waves
    for (int o = 32; o >= tc; o >>= 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { s0[j] += __shfl_xor(s0[j], o, 64); s1[j] += __shfl_xor(s1[j], o, 64); }
    }
    const int lane = tid & 63, wave = tid >> 6;
    if (lane < tc) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { red[(wave * tc + lane) * 16 + j] = s0[j]; red[(wave * tc + lane) * 16 + 8 + j] = s1[j]; }
    }
    __syncthreads();
    for (int t = tid; t < tc * 16; t += 256) {
        const float s = (red[t] + red[tc * 16 + t]) + (red[2 * tc * 16 + t] + red[3 * tc * 16 + t]);
        const int ch = (blockIdx.y * tc + (t >> 4)) * 8 + (t & 7);
        if (ch < g.ld) part[((int64_t)blockIdx.x * 2 + ((t >> 3) & 1)) * g.ld + ch] = s;      // (zeros behind the last channel)
    }
}

// Four channels a workgroup, a thread per partial row: totals, parameter gradients, and the coefficients a, b, c of dx.  The partial sums
// were written from all over the card: few workgroups with long chains of such reads cost 19 us for 1024 rows of 256 channels, this 7 us.
__global__ __launch_bounds__(256) void mx_bn_finish_kernel(const float* __restrict__ part, int groups, int C, int ld, float inv_rows,
                                                           const float* __restrict__ gamma, const float* __restrict__ invstd,
                                                           float* __restrict__ coef, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                           int accumulate) {
    __shared__ float red[4][8];
    const int tid = threadIdx.x, c0 = blockIdx.x * 4;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};       // sums of d, of d (x8 - mean), four channels each
#pragma unroll 4
    for (int g = tid; g < groups; g += 256) {
        const float* p = part + (int64_t)g * 2 * ld + c0;
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p), b = *reinterpret_cast<const u32x4_t*>(p + ld);
#pragma unroll
        for (int j = 0; j < 4; ++j) { s[j] += __uint_as_float(a[j]); s[4 + j] += __uint_as_float(b[j]); }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = wave_sum(s[j]);
    if ((tid & 63) == 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) red[tid >> 6][j] = s[j];
    __syncthreads();
    const int ch = c0 + tid;
    if (tid < 4 && ch < C) {
        const float s0 = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
        const float s1 = (red[0][4 + tid] + red[1][4 + tid]) + (red[2][4 + tid] + red[3][4 + tid]);
        const float is = invstd[ch], dg = s1 * is, a = gamma[ch] * is;
        coef[ch] = a;
        coef[ld + ch] = a * is * dg * inv_rows;
        coef[2 * ld + ch] = a * s0 * inv_rows;
        dgamma[ch] = accumulate ? dgamma[ch] + dg : dg;
        dbeta[ch] = accumulate ? dbeta[ch] + s0 : s0;
    }
}

// what the finish pass leaves, or what the apply pass needs to do its work itself (few groups: a launch costs more than the repeated sums)
struct MxBnTail {
    const float* coef;
    const float* part;
    const float* gamma;
    const float* invstd;
    float* dgamma;
    float* dbeta;
    float inv_rows;
    int groups, accumulate;
};

template <typename T, bool SIGNS, bool FULL, bool JOIN>
__global__ __launch_bounds__(256) void mx_bn_apply_kernel(const MxBnGeom g, const float* __restrict__ mean, const MxBnTail t,
                                                          T* __restrict__ dx, T* __restrict__ dres, const T* __restrict__ racc) {
    const int tid = threadIdx.x, tc = 1 << g.lg, cl = tid & (tc - 1), rl = tid >> g.lg, nrl = 256 >> g.lg;
    const int c = blockIdx.y * tc + cl, left = g.C - c * 8;
    if (left <= 0) return;
    const int64_t r0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * g.per, r1 = r0 + g.per < g.rows ? r0 + g.per : g.rows;
    float ka[8], kb[8], kc[8], mu[8];
    auto get = [&](const float* p, float (&o)[8]) {
        MxRaw8<float> k;
        k.template load<FULL>(p, c * 8, left, true, g.C);
        k.template fix<FULL>();
        k.get(o);
    };
    auto whole = [&](const float* p, float (&o)[8]) {             // a row of `ld` channels (16-byte aligned)
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p + c * 8), b = *reinterpret_cast<const u32x4_t*>(p + c * 8 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] = __uint_as_float(a[j]); o[4 + j] = __uint_as_float(b[j]); }
    };
    get(mean, mu);
    if (JOIN) {
        float s0[8], s1[8], is[8], ga[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { s0[j] = 0.f; s1[j] = 0.f; }
#pragma unroll 4
        for (int k = 0; k < t.groups; ++k) {
            float a[8], b[8];
            whole(t.part + (int64_t)k * 2 * g.ld, a);
            whole(t.part + ((int64_t)k * 2 + 1) * g.ld, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) { s0[j] += a[j]; s1[j] += b[j]; }
        }
        get(t.invstd, is);
        get(t.gamma, ga);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float dg = s1[j] * is[j];
            ka[j] = ga[j] * is[j];
            kb[j] = ka[j] * is[j] * dg * t.inv_rows;
            kc[j] = ka[j] * s0[j] * t.inv_rows;
            if (blockIdx.x == 0 && rl == 0 && j < left) {
                t.dgamma[c * 8 + j] = t.accumulate ? t.dgamma[c * 8 + j] + dg : dg;
                t.dbeta[c * 8 + j] = t.accumulate ? t.dbeta[c * 8 + j] + s0[j] : s0[j];
            }
        }
    } else {
        whole(t.coef, ka);
        whole(t.coef + g.ld, kb);
        whole(t.coef + 2 * g.ld, kc);
    }
    for (int64_t r = r0 + rl; r < r1; r += MXBN_U * nrl) {
        MxBnRow<T> row[MXBN_U];
#pragma unroll
        for (int u = 0; u < MXBN_U; ++u) row[u].template load<SIGNS, FULL>(g, r + u * nrl, c, left, r + u * nrl < r1);
        MX_LOADS_OUT();
#pragma unroll
        for (int u = 0; u < MXBN_U; ++u) {
            if (r + u * nrl < r1) {
                float d[8], v[8], o[8];
                row[u].template get<SIGNS, FULL>(d, v);
                const int64_t at = (r + u * nrl) * g.C + c * 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = fmaf(ka[j], d[j], -fmaf(kb[j], v[j] - mu[j], kc[j]));
                mx_store8f<FULL>(dx + at, left, o);
                if (dres) {
                    if (racc) {
                        mx_load8(racc + at, left, o);
#pragma unroll
                        for (int j = 0; j < 8; ++j) d[j] += o[j];
                    }
                    mx_store8f<FULL>(dres + at, left, d);
                }
            }
        }
    }
}

// Few rows: everything in one launch.  A thread keeps its U rows of a chunk in registers between the sums and dx, so a workgroup (all
// rows of four chunks) reads its inputs once.  The chunks of a cache line belong to neighbouring workgroups: these are dealt to one XCD.
template <typename T, bool SIGNS, bool FULL, int U, int NT>
__global__ __launch_bounds__(NT) void mx_bn_small_kernel(const MxBnGeom g, const float* __restrict__ mean, const MxBnTail t,
                                                         T* __restrict__ dx, T* __restrict__ dres, const T* __restrict__ racc, int wgs) {
    constexpr int TC = 4, nrl = NT / TC, NW = NT / 64;
    __shared__ float red[NW][TC * 16];
    const int per = (wgs + 7) / 8, wg = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (wg >= wgs) return;                                        // (the grid is 8 x per)
    const int tid = threadIdx.x, cl = tid & (TC - 1), rl = tid / TC;
    const int c = wg * TC + cl, left = g.C - c * 8;
    MxBnRow<T> row[U];
    float mu[8], s0[8], s1[8];
    auto get = [&](const float* p, float (&o)[8]) {
        MxRaw8<float> k;
        k.template load<FULL>(p, c * 8, left, true, g.C);
        k.template fix<FULL>();
        k.get(o);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) row[u].template load<SIGNS, FULL>(g, rl + u * nrl, left > 0 ? c : 0, left, left > 0 && rl + u * nrl < g.rows);
    MX_LOADS_OUT();
    get(mean, mu);
#pragma unroll
    for (int j = 0; j < 8; ++j) { s0[j] = 0.f; s1[j] = 0.f; }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (rl + u * nrl < g.rows) {
            float d[8], v[8];
            row[u].template get<SIGNS, FULL>(d, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) { s0[j] += d[j]; s1[j] = fmaf(d[j], v[j] - mu[j], s1[j]); }
        }
    }
    // sixteen lanes hold a chunk's sixteen sums each: every step adds half of what is left over a pair of lanes (15 moves, not 64)
    float r8[8], r4[4], r2[2];
    const bool b5 = tid & 32, b4 = tid & 16, b3 = tid & 8, b2 = tid & 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) r8[j] = (b5 ? s1[j] : s0[j]) + __shfl_xor(b5 ? s0[j] : s1[j], 32, 64);
#pragma unroll
    for (int j = 0; j < 4; ++j) r4[j] = (b4 ? r8[4 + j] : r8[j]) + __shfl_xor(b4 ? r8[j] : r8[4 + j], 16, 64);
#pragma unroll
    for (int j = 0; j < 2; ++j) r2[j] = (b3 ? r4[2 + j] : r4[j]) + __shfl_xor(b3 ? r4[j] : r4[2 + j], 8, 64);
    const float r1 = (b2 ? r2[1] : r2[0]) + __shfl_xor(b2 ? r2[0] : r2[1], 4, 64);
    red[tid >> 6][cl * 16 + (b5 ? 8 : 0) + (b4 ? 4 : 0) + (b3 ? 2 : 0) + (b2 ? 1 : 0)] = r1;
    __syncthreads();
    if (tid < TC * 16) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += red[w][tid];
        red[0][tid] = v;                                          // (each thread has its own column)
    }
    __syncthreads();
    if (left <= 0) return;
    float is[8], ga[8], ka[8], kb[8], kc[8];
    get(t.invstd, is);
    get(t.gamma, ga);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t0 = red[0][cl * 16 + j], t1 = red[0][cl * 16 + 8 + j];
        const float dg = t1 * is[j];
        ka[j] = ga[j] * is[j];
        kb[j] = ka[j] * is[j] * dg * t.inv_rows;
        kc[j] = ka[j] * t0 * t.inv_rows;
        if (rl == 0 && j < left) {
            t.dgamma[c * 8 + j] = t.accumulate ? t.dgamma[c * 8 + j] + dg : dg;
            t.dbeta[c * 8 + j] = t.accumulate ? t.dbeta[c * 8 + j] + t0 : t0;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t r = rl + u * nrl;
        if (r < g.rows) {
            float d[8], v[8], o[8];
            row[u].template get<SIGNS, true>(d, v);               // (put right above)
            const int64_t at = r * g.C + c * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = fmaf(ka[j], d[j], -fmaf(kb[j], v[j] - mu[j], kc[j]));
            mx_store8f<FULL>(dx + at, left, o);
            if (dres) {
                if (racc) {
                    mx_load8(racc + at, left, o);
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] += o[j];
                }
                mx_store8f<FULL>(dres + at, left, d);
            }
        }
    }
}

// a value as it is stored: what rounds to zero is not positive
__device__ static inline float mx_stored(float v, const float*) { return v; }
__device__ static inline float mx_stored(float v, const bf16_t*) { return bf2f(f2bf(v)); }

// Forward: y = act(x scale + shift (+ residual)) and x's checkpoint in one pass (separately the checkpoint reads x and y again).  A thread
// owns eight channels, filler included, and walks rows with its coefficients in registers; a quad of lanes is one block of 32.  Bound by
// memory: 262144 x 256 bf16 with ReLU 70 us (346 MB, 4.9 TB/s), apply and checkpoint apart 103; 65536 x 64 7.3 | 12.0.
template <typename T, bool RES, bool RELU, bool FULL>
__global__ __launch_bounds__(256) void mx_scale_shift_act_kernel(const MxBnGeom g, const T* __restrict__ x, const T* __restrict__ res,
                                                                 const float* __restrict__ scale, const float* __restrict__ shift,
                                                                 T* __restrict__ y, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                 uint8_t* __restrict__ signs) {
    const int tid = threadIdx.x, tc = 1 << g.lg, cl = tid & (tc - 1), rl = tid >> g.lg, nrl = 256 >> g.lg;
    const int c = blockIdx.y * tc + cl, left = g.C - c * 8;
    if (c >= g.cpr) return;                                       // (whole quads: cpr and tc are multiples of four)
    const int64_t r0 = (int64_t)blockIdx.x * g.per, r1 = r0 + g.per < g.rows ? r0 + g.per : g.rows;
    float sc[8], sh[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { sc[j] = j < left ? scale[c * 8 + j] : 0.f; sh[j] = j < left ? shift[c * 8 + j] : 0.f; }
    for (int64_t r = r0 + rl; r < r1; r += MXBN_U * nrl) {
        MxRaw8<T> v[MXBN_U], w[RES ? MXBN_U : 1];
#pragma unroll
        for (int u = 0; u < MXBN_U; ++u) {
            const int64_t at = (r + u * nrl) * g.C + c * 8;
            v[u].template load<FULL>(x, at, left, r + u * nrl < r1, g.C);
            if (RES) w[u].template load<FULL>(res, at, left, r + u * nrl < r1, g.C);
        }
        MX_LOADS_OUT();
#pragma unroll
        for (int u = 0; u < MXBN_U; ++u) {
            const int64_t row = r + u * nrl;
            if (row < r1) {                                       // (a quad's lanes have the same row)
                v[u].template fix<FULL>();
                const uint32_t b = mx_scale_byte<CN_MX_E4M3>(quad_max_u(v[u].absmax()));
                float f[8], o[8];
                v[u].get(f);
                const int64_t i = row * g.cpr + c;
                reinterpret_cast<uint2*>(codes)[i] = mx_codes_e4m3(f, b);
                if ((c & 3) == 0) scales[i >> 2] = (uint8_t)b;
                if (RES) {
                    w[u].template fix<FULL>();
                    w[u].get(o);
                }
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    f[j] = fmaf(f[j], sc[j], sh[j]);
                    if (RES) f[j] += o[j];
                    if (RELU) {
                        f[j] = fmaxf(f[j], 0.f);
                        m |= (mx_stored(f[j], (const T*)nullptr) > 0.f ? 1u : 0u) << j;
                    }
                }
                mx_store8f<FULL>(y + row * g.C + c * 8, left, f);
                if (RELU) signs[i] = (uint8_t)m;
            }
        }
    }
}

// rows of four chunks that a workgroup holds.  us, one launch | two or three: 128x512 5.3 | 10, 512x512 7.1 | 11, 700x512 8.3 | 11.6; eight rows
// a thread for 2048 rows: 1471x30 16 | 10.2.  Threads and rows of one: 128x512 in 256 threads 5.3, in 1024 5.6; 512x2048 with two rows 7.6,
// with four 7.8
#define MXBN_SMALL 1024

static int mxbn_lg(int C) {
    const int chunks = cdiv(C, 8);
    int lg = 0;
    while (lg < 5 && (1 << lg) < chunks) ++lg;
    return lg;
}
// row groups up to which the apply pass adds the partial sums up itself: a launch less for the host (3 us there), and little more on the
// device (4515x28 11.7 us, 10.9 with a finish pass; up to 128 groups 4096x256 would take 39 instead of 11.4)
#define MXBN_JOIN 32
// row groups of the sums pass: ~512 workgroups in all, at least four rows for a thread.  us, 256 | 512 | 1024 | 2048 workgroups: 262144x256
// 118 | 106 | 111 | 116, 1048576x64 118 | 106 | 108 | 112, 16384x512 21.3 | 21.6 | 23.7 | 23.7
static int mxbn_groups(int64_t rows, int C) {
    const int lg = mxbn_lg(C), tiles = cdiv(cdiv(C, 8), 1 << lg);
    const int64_t most = (rows + 4 * (256 >> lg) - 1) / (4 * (256 >> lg));
    int64_t g = 512 / tiles;
    g = g < most ? g : most;
    return (int)(g < 1 ? 1 : g);
}

extern "C" size_t cn_mx_bn_bwd_bytes(int64_t rows, int C, int dtype) {
    if (rows <= MXBN_SMALL || C < 1 || C > MX_MAX_C) return 0;
    return sizeof(float) * ((size_t)mxbn_groups(rows, C) * 2 + 3) * (size_t)(cdiv(C, 8) * 8);
}

extern "C" int cn_mx_bn_bwd(const void* dy, const void* codes, const void* scales, const void* signs, const float* gamma, const float* mean,
                            const float* invstd, void* dx, void* dres, const void* racc, float* dgamma, float* dbeta, int accumulate,
                            int64_t rows, int C, int dtype, void* ws, size_t ws_bytes, void* stream) {
    CN_CHECK_ARG(rows >= 1 && C >= 1 && C <= MX_MAX_C && rows <= ((int64_t)1 << 40) / C, "cn_mx_bn_bwd: rows %lld, channels %d", (long long)rows, C);
    CN_CHECK_ARG(dtype == CN_F32 || dtype == CN_BF16, "cn_mx_bn_bwd: bad dtype %d", dtype);
    CN_CHECK_ARG(dy && codes && scales && gamma && mean && invstd && dx && dgamma && dbeta, "cn_mx_bn_bwd: null pointer");
    CN_CHECK_ARG(dres || !racc, "cn_mx_bn_bwd: racc without dres");
    CN_CHECK_ARG(((uintptr_t)codes & 15) == 0, "cn_mx_bn_bwd: codes must be 16-byte aligned");
    CN_CHECK_ARG(((uintptr_t)ws & 15) == 0, "cn_mx_bn_bwd: the workspace must be 16-byte aligned");
    if (ws_bytes < cn_mx_bn_bwd_bytes(rows, C, dtype) || (!ws && ws_bytes)) {
        cn_set_error("cn_mx_bn_bwd: workspace of %zu bytes needed", cn_mx_bn_bwd_bytes(rows, C, dtype));
        return CN_EWORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    const bool full = C % 8 == 0;
#define MXBN_GO(KERNEL, MORE, GRID, ...)                                                                                               \
    CN_DISPATCH_DTYPE(dtype, T, {                                                                                                      \
        if (signs) { if (full) KERNEL<T, true, true MORE><<<GRID, 256, 0, st>>>(__VA_ARGS__); else KERNEL<T, true, false MORE><<<GRID, 256, 0, st>>>(__VA_ARGS__); }  \
        else { if (full) KERNEL<T, false, true MORE><<<GRID, 256, 0, st>>>(__VA_ARGS__); else KERNEL<T, false, false MORE><<<GRID, 256, 0, st>>>(__VA_ARGS__); }      \
    })
#define MXBN_COMMA ,
    if (rows <= MXBN_SMALL) {
        const MxBnGeom g{dy, (const uint8_t*)codes, (const uint8_t*)scales, (const uint8_t*)signs, rows, C, cdiv(C, MX_BLOCK) * 4, cdiv(C, MX_BLOCK), 0, 0, 0};
        const MxBnTail t{nullptr, nullptr, gamma, invstd, dgamma, dbeta, 1.f / (float)rows, 0, accumulate};
        const int wgs = cdiv(cdiv(C, 8), 4), grid = cdiv(wgs, 8) * 8;
#define MXBN_SMALL_GO(T, S, U, NT)                                                                                                     \
    do { if (full) mx_bn_small_kernel<T, S, true, U, NT><<<grid, NT, 0, st>>>(g, mean, t, (T*)dx, (T*)dres, (const T*)racc, wgs);      \
         else mx_bn_small_kernel<T, S, false, U, NT><<<grid, NT, 0, st>>>(g, mean, t, (T*)dx, (T*)dres, (const T*)racc, wgs); } while (0)
#define MXBN_SMALL_ROWS(T, S)                                                                                                          \
    do { if (rows <= 128) MXBN_SMALL_GO(T, S, 2, 256); else if (rows <= 512) MXBN_SMALL_GO(T, S, 2, 1024); else MXBN_SMALL_GO(T, S, 4, 1024); } while (0)
        if (dtype == CN_BF16) { if (signs) MXBN_SMALL_ROWS(bf16_t, true); else MXBN_SMALL_ROWS(bf16_t, false); }
        else { if (signs) MXBN_SMALL_ROWS(float, true); else MXBN_SMALL_ROWS(float, false); }
#undef MXBN_SMALL_ROWS
#undef MXBN_SMALL_GO
        CN_LAUNCH_CHECK("cn_mx_bn_bwd");
        return CN_OK;
    }
    const int groups = mxbn_groups(rows, C);
    float* part = (float*)ws;
    const int ld = cdiv(C, 8) * 8;
    float* coef = part + (size_t)groups * 2 * ld;
    MxBnGeom g{dy, (const uint8_t*)codes, (const uint8_t*)scales, (const uint8_t*)signs, rows, C, cdiv(C, MX_BLOCK) * 4, cdiv(C, MX_BLOCK), ld, mxbn_lg(C), 0};
    const int tiles = cdiv(cdiv(C, 8), 1 << g.lg);
    const int nrl = 256 >> g.lg;
    CN_CHECK_ARG(tiles <= 65535, "cn_mx_bn_bwd: too many channels");
    // apply pass: eight rows a thread (its coefficients are loaded once), fewer where that would leave less than two workgroups a compute unit (us, this
    // rule | always two rows | always eight: 4515x28 11.7 | 12.0 | 14.7, 8192x256 13.2 | 13.2 | 14.1, 262144x256 110 | 113 | 110)
    int deep = 8;
    while (deep > 1 && (rows + deep * nrl - 1) / (deep * nrl) * tiles < 512) deep /= 2;
    g.per = (int64_t)deep * nrl;
    CN_CHECK_ARG(mx_grid_fits((rows + g.per - 1) / g.per, 256), "cn_mx_bn_bwd: too many rows for one launch");
    MXBN_GO(mx_bn_sums_kernel, , dim3(groups, tiles), g, mean, part);
    CN_LAUNCH_CHECK("cn_mx_bn_bwd");
    const MxBnTail t{coef, part, gamma, invstd, dgamma, dbeta, 1.f / (float)rows, groups, accumulate};
    const bool joined = groups <= MXBN_JOIN;
    if (!joined) {
        mx_bn_finish_kernel<<<cdiv(C, 4), 256, 0, st>>>(part, groups, C, ld, t.inv_rows, gamma, invstd, coef, dgamma, dbeta, accumulate);
        CN_LAUNCH_CHECK("cn_mx_bn_bwd");
    }
    const int ng = cdiv(rows, g.per);
    if (joined) MXBN_GO(mx_bn_apply_kernel, MXBN_COMMA true, dim3(ng, tiles), g, mean, t, (T*)dx, (T*)dres, (const T*)racc);
    else MXBN_GO(mx_bn_apply_kernel, MXBN_COMMA false, dim3(ng, tiles), g, mean, t, (T*)dx, (T*)dres, (const T*)racc);
#undef MXBN_GO
#undef MXBN_COMMA
    CN_LAUNCH_CHECK("cn_mx_bn_bwd");
    return CN_OK;
}

extern "C" int cn_mx_scale_shift_act(const void* x, const void* residual, const float* scale, const float* shift, void* y, void* codes,
                                     void* scales, void* signs, int64_t rows, int C, int relu, int dtype, void* stream) {
    CN_CHECK_ARG(rows >= 0 && C >= 1 && C <= MX_MAX_C && rows <= ((int64_t)1 << 40) / C, "cn_mx_scale_shift_act: rows %lld, channels %d", (long long)rows, C);
    CN_CHECK_ARG(dtype == CN_F32 || dtype == CN_BF16, "cn_mx_scale_shift_act: bad dtype %d", dtype);
    if (rows == 0) return CN_OK;                                  // (an empty buffer's pointers are null)
    CN_CHECK_ARG((signs != nullptr) == (relu != 0), "cn_mx_scale_shift_act: signs come with relu");
    CN_CHECK_ARG(x && scale && shift && y && codes && scales, "cn_mx_scale_shift_act: null pointer");
    CN_CHECK_ARG(((uintptr_t)codes & 15) == 0, "cn_mx_scale_shift_act: codes must be 16-byte aligned");
    MxBnGeom g{nullptr, nullptr, nullptr, nullptr, rows, C, cdiv(C, MX_BLOCK) * 4, cdiv(C, MX_BLOCK), 0, 2, 0};
    while (g.lg < 5 && (1 << g.lg) < g.cpr) ++g.lg;
    const int tiles = cdiv(g.cpr, 1 << g.lg), nrl = 256 >> g.lg;
    int deep = 8;                                                 // rows a thread, by the backward pass's rule
    while (deep > 1 && (rows + deep * nrl - 1) / (deep * nrl) * tiles < 512) deep /= 2;
    g.per = (int64_t)deep * nrl;
    CN_CHECK_ARG(mx_grid_fits((rows + g.per - 1) / g.per, 256), "cn_mx_scale_shift_act: too many rows for one launch");
    const dim3 grid(cdiv(rows, g.per), tiles);
    hipStream_t st = (hipStream_t)stream;
#define MXSS(RES, RELU, FULL)                                                                                                          \
    mx_scale_shift_act_kernel<T, RES, RELU, FULL><<<grid, 256, 0, st>>>(g, (const T*)x, (const T*)residual, scale, shift, (T*)y,       \
                                                                        (uint8_t*)codes, (uint8_t*)scales, (uint8_t*)signs)
#define MXSS_F(RES, RELU) do { if (C % 8 == 0) MXSS(RES, RELU, true); else MXSS(RES, RELU, false); } while (0)
    CN_DISPATCH_DTYPE(dtype, T, {
        if (residual) { if (relu) MXSS_F(true, true); else MXSS_F(true, false); }
        else { if (relu) MXSS_F(false, true); else MXSS_F(false, false); }
    });
#undef MXSS_F
#undef MXSS
    CN_LAUNCH_CHECK("cn_mx_scale_shift_act");
    return CN_OK;
}
