// y = act(x4 @ w4^T + bias + residual): x [M][K] is quantised to e2m1 on the way in (one scale per 32 channels, mx_common.h), w [N][K]
// was quantised and laid out once (cn_mx_pack_weight).  Products of 4-bit values times powers of two are exact, sums are fp32
// (v_mfma_scale_f32_32x32x64_f8f6f4: a lane's 16 bytes are one block of 32 channels, its scale rides in a byte of a register).
//
// What has to move is x in and y out; the codes of x never leave the workgroup.  A workgroup quantises its BM rows once into LDS and
// keeps them there while it walks its columns; the weights stream from L2 in fragment order (1 KB contiguous per 32 columns x 64
// channels).  With 1024 row tiles or more a workgroup walks all columns and x is read and quantised once whatever N is (65536x1024x256:
// 129.5 MiB read for 128 MiB of x); fewer row tiles share their columns out to as many workgroups as fill the card, and each of these reads
// and quantises the rows again.  K beyond what LDS holds (7936 channels; 7872 and 6784 with four and eight waves over the channels) is taken in chunks, and
// then every 256 columns (32 with waves over the channels) read and quantise x again: 4096x9000x2048 does so eight times.
// Bound by memory: 65536x256x1024 with its residual 57 us (302 MB, 5.3 TB/s, the rate of a copy), 65536x1024x256 41 us (168 MB, 4.1 TB/s:
// reading x alone takes 28, quantising, products and stores overlap with it in part), 1x2048x512 4.2 us (latency of one row's K).
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
    int K, N, S, S4;           // S: steps of 64 channels, S4 = ceil(S / 4) groups
    int t32;                   // 32-column tiles in all
    int chunk;                 // steps that LDS holds (a multiple of 4 unless it is S)
    int per_wg;                // passes over the workgroup's columns
    int relu;
    int pitch, spitch;         // LDS bytes per row: codes, scales
    int sc_ofs, ep_ofs;        // LDS offsets of the scales and of the output staging
};

// two steps of NJ weight tiles
template <int NJ> struct MxLinB { u32x4_t f[2][NJ]; };

// 32 x 32 NJ outputs per wave; WM x WN waves over rows and columns, or WK over the channels (few rows: the launch would be short of waves
// otherwise; their sums meet in LDS, in a fixed order).  resident: LDS holds all K channels of the rows.  RT > 1 (K <= 256): a wave takes
// RT row tiles one after the other with the weights of its columns in registers (read from L2 half as often: 65536x256x1024 69 -> 63 us).
// Held to four waves a SIMD (128 registers) in 16 bits, that form spills 1 - 3 of them for even K and 8 for ragged ones.
template <typename T, int RT, int NJ, int WM, int WN, int WK, bool FULLK, bool FULLN, bool resident>
__global__ __launch_bounds__(64 * WM * WN * WK, resident && sizeof(T) == 2 ? 4 : 2) void mx_linear_kernel(const MxLinGeom g) {
    static_assert((WK == 1 ? WM * WN == 4 : WM * WN == 1) && (RT == 1 || (WK == 1 && resident)), "rows and columns, or channels");
    constexpr int NT = 64 * WM * WN * WK;
    constexpr int BM = 32 * RT * WM, EPN = 32 * NJ, EPP = EPN + 4;         // EPP: floats per staged output row (rows on different banks)
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = WK > 1 ? 0 : wave / WN, wn = WK > 1 ? 0 : wave % WN, wk = WK > 1 ? wave : 0;
    const int64_t m0 = (int64_t)blockIdx.x * BM;
    const int rows = (int)(g.M - m0 < BM ? g.M - m0 : BM);
    const T* __restrict__ X = reinterpret_cast<const T*>(g.x) + m0 * g.K;

    // Quantise channels 64 s0 .. 64 s1 of the workgroup's rows into LDS (rows behind the last stay as they are: what they give is not
    // stored).  A thread's chunks are NT apart; row and channel are carried along (multiplications cost four times an addition).
    auto stage = [&](int s0, int s1) {
        const int d = (s1 - s0) * 8, dq = NT / d, dr = NT - dq * d;          // 8-channel chunks per row (uniform)
        const uint32_t step = (uint32_t)(dq * g.K + dr * 8), wrap = (uint32_t)(g.K - d * 8);
        constexpr int U = sizeof(T) == 2 && WK == 1 ? 8 : 4;                   // loads in flight per thread; WK > 1: and as many again
        struct At { int row, pc; uint32_t ofs; };
        auto next = [&](At& t) {
            t.row += dq;
            t.pc += dr;
            t.ofs += step;
            if (t.pc >= d) { t.pc -= d; t.row += 1; t.ofs += wrap; }
        };
        struct Batch { MxRaw8<T> v[U]; };
        auto ask = [&](Batch& q, At& t) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                q.v[u].template load<FULLK>(X, t.ofs, g.K - s0 * 64 - t.pc * 8, t.row < rows, g.K);
                next(t);
            }
            MX_LOADS_OUT();
        };
        auto take = [&](Batch& q, At& t) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                q.v[u].template fix<FULLK>();
                const uint32_t b = mx_scale_byte<CN_MX_E2M1>(quad_max_u(q.v[u].absmax()));
                if (t.row < rows) {                               // (whole quads)
                    *reinterpret_cast<uint32_t*>(smem + t.row * g.pitch + t.pc * 4) = q.v[u].codes_e2m1(b);
                    const int blk = t.pc >> 2, s = blk >> 1;      // byte s & 3 of word (s / 4, half)
                    if ((t.pc & 3) == 0) smem[g.sc_ofs + t.row * g.spitch + ((s >> 2) * 2 + (blk & 1)) * 4 + (s & 3)] = (uint8_t)b;
                }
                next(t);
            }
        };
        At t0;
        t0.row = tid / d;
        t0.pc = tid - t0.row * d;
        t0.ofs = (uint32_t)(t0.row * g.K + s0 * 64 + t0.pc * 8);
        At t1 = t0;
        if (WK == 1) {
            while (t1.row < rows) {
                Batch q;
                ask(q, t0);
                take(q, t1);
            }
        } else {
            Batch q, r;
            ask(q, t0);
            while (t1.row < rows) {
                if (t0.row < rows) ask(r, t0);
                take(q, t1);
                if (t1.row < rows) {
                    if (t0.row < rows) ask(q, t0);
                    take(r, t1);
                }
            }
        }
    };
    // steps s, s + 1 and the scales of their group for the columns of pass `it` (beyond the last: a readable address, not used)
    auto loadb = [&](MxLinB<NJ>& B, int it, int s) {
        const int first = ((blockIdx.y * g.per_wg + it) * WN + wn) * NJ;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int nt = first + j < g.t32 ? first + j : g.t32 - 1;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int q = s + u < g.S ? s + u : g.S - 1;
                // (a uniform base and a lane offset: no address registers; the index stays below 2^28)
                B.f[u][j] = reinterpret_cast<const u32x4_t*>(g.wc + __builtin_amdgcn_readfirstlane((nt * g.S + q) * 64))[lane];
            }
        }
    };
    auto loads = [&](uint32_t (&q)[NJ], int it, int t) {
        const int first = ((blockIdx.y * g.per_wg + it) * WN + wn) * NJ;
        t = t < g.S4 ? t : g.S4 - 1;
#pragma unroll
        for (int j = 0; j < NJ; ++j) q[j] = (g.ws + __builtin_amdgcn_readfirstlane(((first + j < g.t32 ? first + j : g.t32 - 1) * g.S4 + t) * 64))[lane];
    };
    f32x16_t acc[NJ];
    const unsigned char* arow = smem + (wm * RT * 32 + (lane & 31)) * g.pitch + (lane >> 5) * 16;
    const unsigned char* srow = smem + g.sc_ofs + (wm * RT * 32 + (lane & 31)) * g.spitch + (lane >> 5) * 4;
    // step s + u of row tile i (byte U of the scale words)
#define MXL_STEP(B, u, U)                                                                                                               \
    if (s + u < s1) {                                                                                                                   \
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(arow + i * 32 * g.pitch + (s + u - s0) * 32);                               \
        const i32x8_t av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};                                                        \
        _Pragma("unroll") for (int j = 0; j < NJ; ++j) {                                                                                \
            const i32x8_t bv = {(int)B.f[u][j].x, (int)B.f[u][j].y, (int)B.f[u][j].z, (int)B.f[u][j].w, 0, 0, 0, 0};                    \
            acc[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc[j], 4, 4, U, (int)sa, U, (int)sb[j]);                  \
        }                                                                                                                               \
    }
    // eight finished columns of a row; rv: the residual input there (zeros: none)
    auto finish = [&](float (&v)[8], MxRaw8<T>& rv, int64_t m, int nc, int left, const float (&bs)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bs[e];
        if (g.res) {
            float r[8];
            rv.template fix<FULLN>();
            rv.get(r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        if (g.relu) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];            // (a NaN stays one)
        }
        if (m < g.M) mx_store8f<FULLN>(reinterpret_cast<T*>(g.y) + m * g.N + nc, left, v);
    };

    MxLinB<NJ> B0, B1;
    uint32_t sb[NJ];
    if (resident) {
        loadb(B0, 0, 4 * wk);                                     // in flight while the rows are quantised
        if (RT > 1) loadb(B1, 0, 2);
        loads(sb, 0, wk);
        stage(0, g.S);
        __syncthreads();
    }
    constexpr int LPR = EPN / 8, RPI = 64 / LPR, NQ = 16 / RPI;   // lanes per staged row, rows per wave instruction, instructions per 16 rows
    for (int it = 0; it < g.per_wg; ++it) {
        const int n0 = ((blockIdx.y * g.per_wg + it) * WN + wn) * EPN;
        if (resident && WK == 1 && n0 >= g.N) break;              // (no barrier below in that form)
        const int nl = WK > 1 ? tid % LPR : lane % LPR, nc = n0 + nl * 8, left = g.N - nc;
#pragma unroll 1
        for (int i = 0; i < RT; ++i) {
            const int64_t mt = m0 + (wm * RT + i) * 32;
            // the residual rows are asked for before the products: their latency is the longest here
            MxRaw8<T> rv[WK == 1 ? 2 * NQ : 1];
            if (WK == 1 && g.res) {
#pragma unroll
                for (int q = 0; q < 2 * NQ; ++q) {
                    const int64_t m = mt + q * RPI + lane / LPR;
                    rv[q].template load<FULLN>(reinterpret_cast<const T*>(g.res), m * g.N + nc, left, m < g.M, g.N);
                }
                MX_LOADS_OUT();
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
            if (RT > 1) {
                constexpr int s0 = 0;
                const int s1 = g.S;
                const uint32_t sa = *reinterpret_cast<const uint32_t*>(srow + i * 32 * g.spitch);
                int s = 0;
                MXL_STEP(B0, 0, 0) MXL_STEP(B0, 1, 1)
                s = 2;
                MXL_STEP(B1, 0, 2) MXL_STEP(B1, 1, 3)
                if (i == RT - 1 && it + 1 < g.per_wg) {
                    loadb(B0, it + 1, 0);
                    loadb(B1, it + 1, 2);
                    loads(sb, it + 1, 0);
                }
            } else {
                for (int s0 = 0; s0 < g.S; s0 += resident ? g.S : g.chunk) {
                    const int s1 = resident || s0 + g.chunk > g.S ? g.S : s0 + g.chunk;
                    int s = s0 + 4 * wk;
                    if (!resident) {
                        __syncthreads();
                        loadb(B0, it, s);
                        loads(sb, it, s >> 2);
                        stage(s0, s1);
                        __syncthreads();
                    }
                    for (; s < s1; s += 4 * WK) {
                        const uint32_t sa = *reinterpret_cast<const uint32_t*>(srow + ((s - s0) >> 2) * 8);
                        uint32_t sn[NJ];
                        loadb(B1, it, s + 2);
                        loads(sn, it, (s >> 2) + WK);
                        MXL_STEP(B0, 0, 0) MXL_STEP(B0, 1, 1)
                        loadb(B0, it, s + 4 * WK);
                        s += 2;
                        MXL_STEP(B1, 0, 2) MXL_STEP(B1, 1, 3)
                        s -= 2;
#pragma unroll
                        for (int j = 0; j < NJ; ++j) sb[j] = sn[j];
                    }
                }
                if (resident && it + 1 < g.per_wg) {
                    loadb(B0, it + 1, 4 * wk);
                    loads(sb, it + 1, wk);
                }
            }
            float bs[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) bs[e] = 0.f;
            if (g.bias) {
                MxRaw8<float> b;
                b.template load<FULLN>(g.bias, nc, left, true, g.N);
                b.template fix<FULLN>();
                b.get(bs);
            }
            if (WK == 1) {
                // 16 rows at a time through the wave's own slice of LDS, then eight columns a lane
                float* ep = reinterpret_cast<float*>(smem + g.ep_ofs) + wave * 16 * EPP;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e) ep[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * EPP + j * 32 + (lane & 31)] = acc[j][8 * h + e];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        const int r = q * RPI + lane / LPR;
                        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(ep + r * EPP + nl * 8), hi = *reinterpret_cast<const f32x4_t*>(ep + r * EPP + nl * 8 + 4);
                        float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                        finish(v, rv[h * NQ + q], mt + h * 16 + r, nc, left, bs);
                    }
                }
            } else {
                float* ep = reinterpret_cast<float*>(smem + g.ep_ofs);
                __syncthreads();
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) ep[(wk * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * EPP + j * 32 + (lane & 31)] = acc[j][e];
                __syncthreads();
                for (int r = tid / LPR; r < rows; r += NT / LPR) {
                    if (g.res) rv[0].template load<FULLN>(reinterpret_cast<const T*>(g.res), (m0 + r) * g.N + nc, left, true, g.N);
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
                    for (int k = 0; k < WK; ++k) {
                        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(ep + (k * 32 + r) * EPP + nl * 8), hi = *reinterpret_cast<const f32x4_t*>(ep + (k * 32 + r) * EPP + nl * 8 + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) { v[e] += lo[e]; v[4 + e] += hi[e]; }
                    }
                    finish(v, rv[0], m0 + r, nc, left, bs);
                }
            }
        }
    }
#undef MXL_STEP
}

// the form of a product: row tiles, 32-column tiles and waves over rows, columns and channels (the kernel's parameters)
struct MxLinForm { int rt, nj, wm, wn, wk; };
// LDS of a workgroup that holds `chunk` steps of its rows: bytes per row, then the output staging
struct MxLinLds { int chunk, pitch, spitch, rows, ep; };
static MxLinLds mxl_lds(const MxLinForm& f, int S) {
    MxLinLds l;
    const int BM = 32 * f.rt * f.wm, EPP = 32 * f.nj + 4;
    l.ep = (f.wk > 1 ? f.wk * 32 : 4 * 16) * EPP * 4;
    l.chunk = S;
    auto bytes = [&](int c) {
        l.pitch = c * 32 + 16;                      // an odd number of 16-byte pieces: eight rows' reads hit different banks
        l.spitch = cdiv(c, 4) * 8 + 4;
        return BM * (l.pitch + l.spitch);
    };
    // all channels of the rows where they fit, else a chunk at a time
    while ((l.rows = bytes(l.chunk)) + l.ep > 150 * 1024) l.chunk = l.chunk > 128 ? 128 : l.chunk / 2 / 4 * 4;
    return l;
}

template <typename T, int RT, int NJ, int WM, int WN, int WK, bool FULLK, bool FULLN>
static int mxl_launch(MxLinGeom g, hipStream_t st) {
    constexpr int BM = 32 * RT * WM;
    constexpr int NT = 64 * WM * WN * WK;
    constexpr bool CHUNKED = RT * WM == 1;                         // (the forms of more rows are for K <= 256, which always fits)
    const MxLinLds l = mxl_lds(MxLinForm{RT, NJ, WM, WN, WK}, g.S);
    const int chunk = l.chunk, ep = l.ep;
    g.chunk = chunk;
    g.pitch = l.pitch;
    g.spitch = l.spitch;
    g.sc_ofs = BM * g.pitch;
    g.ep_ofs = (l.rows + 15) / 16 * 16;
    const int smem = g.ep_ofs + ep;
    g.t32 = cdiv(g.N, 32);
    const int64_t mt = (g.M + BM - 1) / BM;
    CN_CHECK_ARG(mx_grid_fits(mt, NT), "cn_mx_linear_fwd: too many rows for one launch");
    const int passes = cdiv(g.t32, NJ * WN);
    // one workgroup walks all columns of its rows unless that leaves less than four workgroups a compute unit.  us, never split | this rule |
    // one pass a workgroup: 512x512x2048 16.8 | 6.5 | 6.8, 4096x512x2048 19.3 | 13.1 | 13.1, 16384x256x1024 14.8 | 14.9 | 17.1,
    // 65536x256x1024 36.3 | 36.3 | 45.6 (no residual)
    int64_t split = mt >= 1024 ? 1 : (1024 + mt - 1) / mt;
    if (chunk < g.S || split > passes) split = passes;
    g.per_wg = cdiv(passes, split);
    split = cdiv(passes, g.per_wg);
    static bool attr[64] = {};
    int dev = 0;
    CN_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !attr[dev]) {
        CN_HIP(hipFuncSetAttribute((const void*)mx_linear_kernel<T, RT, NJ, WM, WN, WK, FULLK, FULLN, true>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if constexpr (CHUNKED)
            CN_HIP(hipFuncSetAttribute((const void*)mx_linear_kernel<T, RT, NJ, WM, WN, WK, FULLK, FULLN, false>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (dev < 64) attr[dev] = true;
    }
    const dim3 grid((unsigned)mt, (unsigned)split);
    if (!CHUNKED || chunk >= g.S) mx_linear_kernel<T, RT, NJ, WM, WN, WK, FULLK, FULLN, true><<<grid, NT, smem, st>>>(g);
    else if constexpr (CHUNKED) mx_linear_kernel<T, RT, NJ, WM, WN, WK, FULLK, FULLN, false><<<grid, NT, smem, st>>>(g);
    CN_LAUNCH_CHECK("cn_mx_linear_fwd");
    return CN_OK;
}
// Which waves do what, us (bf16, M x K x N):
//   K split over the waves, 32 x 32 a workgroup | columns over the waves, 32 x 256: 64x1440x64 8.8 | 10.3, 512x2048x512 10.9 | 13.0,
//     2048x64x256 5.1 | 5.5, 20000x1440x8 15.4 | 17.5, and there over four | eight waves (one workgroup a compute unit at most and more than
//     16384 values for it to quantise): 41x1872x82 10.7 | 9.1, 256x4096x256 18.4 | 14.4, 1x2048x512 5.0 | 5.0, 8x2048x512 5.8 | 5.6, 32x256x64 4.9 | 5.2, 296x752x1106 8.5 |
//     9.1 (sixteen: 9.1, 13.7, 5.4, 6.0, 11.8); the other way 512x512x2048 9.3 | 6.6, 8192x512x64 6.9 | 6.4, 8192x1024x256 15.2 | 10.0
//   rows over the waves, 128 x 64 | 64 x 128 | 32 x 256: 65536x64x64 7.4 | 8.7 | 11.4, 65536x256x128 16.4 | 13.3 | 14.7, 65536x512x64
//     17.5 | 17.4 | 16.4, 65536x1024x256 111 | 53 | 44
//   32 x 256 | two row tiles, 64 x 256: 65536x256x1024 with its residual 69 | 63, 262144x64x256 52 | 41, 32768x256x512 14.4 | 15.7
static MxLinForm mxl_form(int64_t M, int K, int N) {
    const int64_t wgs = (M + 31) / 32 * cdiv(N, 32);
    if (N <= 32 || wgs <= 512) return wgs <= 256 && (M < 32 ? M : 32) * K > 16384 ? MxLinForm{1, 1, 1, 1, 8} : MxLinForm{1, 1, 1, 1, 4};
    if (N <= 64 && K <= 256) return MxLinForm{1, 2, 4, 1, 1};
    if (N <= 128 && K <= 256) return MxLinForm{1, 2, 2, 2, 1};
    return K <= 256 && M >= 49152 ? MxLinForm{2, 2, 1, 4, 1} : MxLinForm{1, 2, 1, 4, 1};
}
template <typename T, bool FULLK, bool FULLN>
static int mxl_choose(const MxLinGeom& g, hipStream_t st) {
    const MxLinForm f = mxl_form(g.M, g.K, g.N);
    if (f.wk == 8) return mxl_launch<T, 1, 1, 1, 1, 8, FULLK, FULLN>(g, st);
    if (f.wk == 4) return mxl_launch<T, 1, 1, 1, 1, 4, FULLK, FULLN>(g, st);
    if (f.wm == 4) return mxl_launch<T, 1, 2, 4, 1, 1, FULLK, FULLN>(g, st);
    if (f.wm == 2) return mxl_launch<T, 1, 2, 2, 2, 1, FULLK, FULLN>(g, st);
    if (f.rt == 2) return mxl_launch<T, 2, 2, 1, 4, 1, FULLK, FULLN>(g, st);
    return mxl_launch<T, 1, 2, 1, 4, 1, FULLK, FULLN>(g, st);
}

extern "C" int cn_mx_linear_variant(int64_t M, int K, int N) {
    if (M < 1 || K < 1 || N < 1 || K > MX_MAX_C || N > MX_MAX_C) return 0;
    const MxLinForm f = mxl_form(M, K, N);
    const int S = cdiv(K, 64);
    return (mxl_lds(f, S).chunk < S ? 100000 : 0) + f.rt * 10000 + f.nj * 1000 + f.wm * 100 + f.wn * 10 + f.wk;
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
#define MXL_GO(T) do { if (K % 8 == 0) return N % 8 == 0 ? mxl_choose<T, true, true>(g, st) : mxl_choose<T, true, false>(g, st);       \
                       return N % 8 == 0 ? mxl_choose<T, false, true>(g, st) : mxl_choose<T, false, false>(g, st); } while (0)
    if (dtype == CN_BF16) MXL_GO(bf16_t);
    MXL_GO(float);
#undef MXL_GO
}
