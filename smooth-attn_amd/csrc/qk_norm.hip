// RMS norm of each head's query and key rows and rotate-half RoPE, in one
// pass: the step between the projections and the attention.
//
// For a row x of D elements at position t, with the head dim's weight w:
//   r = 1 / sqrt(mean(x^2) + eps),  n = r x,  z = w n,
//   y_d = z_d cos - z_{d+D/2} sin,  y_{d+D/2} = z_{d+D/2} cos + z_d sin
// in fp32, rounded once, to the output's type (the reciprocal root is v_rsq_f32's,
// at most 3/4 of a step off).  Backward, with g = dL/dy:
//   dz_d = g_d cos + g_{d+D/2} sin,  dz_{d+D/2} = g_{d+D/2} cos - g_d sin,
//   dw = sum over rows of dz n,  h = w dz,
//   dx = r (h - n mean(h n)) = r h - r^3 x mean(h x)
// (the second form needs no r before its sum, so both sums of a row are
// reduced together).
//
// Layout.  A lane holds a pair of 8-element chunks (d, d + D/2) of one row,
// so a rotation stays within a lane, and L = D/16 lanes (rounded up to a power
// of two) hold a row; the 64 / L rows of a wave are HG heads of 64 / (L HG)
// tokens.  cos and sin are 32 bits each against 16 for an element, so reading
// them for every row would double the traffic: a wave keeps its tokens' angles
// in registers over all the heads of its chunk.  Where the heads of a token lie
// next to each other in memory ([B, T, H, D] buffers), the rows of a wave are
// heads first, else tokens first, so a wave reads contiguous spans.
//
// The serving form takes packed tokens, each with its position and its slot in
// the paged caches: q is written to a tensor, k and v (v only converted) to
// the caches, each value rounded once to the cache's type.
//
// Bound by memory: [4,32/32,4096,128] bf16 90 us forward and 135 backward (6.0
// TB/s), 8211 tokens of Hq 32 / Hkv 8, D = 128 into e4m3fn caches 40 us (4.7
// TB/s); few tokens by the launch (8 tokens 4.3 us).
#include <algorithm>

#include "common.hpp"

namespace sa {
namespace {

constexpr int kBlockWaves = 4;
constexpr int kCus = 256;

// One of the tensors of a launch: its rows in, and where they go.
struct NormSide {
    const void* x;
    const void* g;  // backward: gradient of the output
    void* y;        // forward: the output; backward: gradient of x
    const void* w;  // nullable: ones
    int64_t xs[3], gs[3], ys[3];  // element strides (b, h, t) (caches: page, h, row)
    int H;
    int cache;  // element type of the caches' rows (serving), else -1
    int norm;   // 0: rows are only converted
};

struct NormParams {
    NormSide side[3];
    const float* cos;
    const float* sin;
    const int32_t* pos;    // nullable: row t of the tables
    const int32_t* slots;  // serving: cache slot of each token, negative for none
    int64_t pos_b;         // batch stride of pos
    float* partial;        // backward: dw of each block
    float eps;
    int first[4];  // first chunk of each side
    int CH;        // heads per chunk
    int logHG;     // log2 of the heads among a wave's rows
    int T, D, n_pos, n_tokens, n_tiles, w32, page_size, n_pages;
};

// 8 consecutive elements.  STREAM: past the caches (see streams()).
template <bool STREAM>
__device__ __forceinline__ u32x4 get16(const void* p) {
    return STREAM ? load16(p) : *static_cast<const u32x4*>(p);
}
template <bool STREAM>
__device__ __forceinline__ void put16(void* p, u32x4 v) {
    if constexpr (STREAM) store16(p, v);
    else *static_cast<u32x4*>(p) = v;
}
template <typename T, bool STREAM = false>
__device__ __forceinline__ void load8(const T* p, float* f) {
    const u32x4 a = get16<STREAM>(p);
    if constexpr (sizeof(T) == 4) {
        const u32x4 b = get16<STREAM>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = __uint_as_float(a[i]);
            f[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = elem<T>(w, i);
    }
}
template <typename T, bool STREAM = false>
__device__ __forceinline__ void store8(T* p, const float* f) {
    if constexpr (sizeof(T) == 4) {
        put16<STREAM>(p, u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                               __float_as_uint(f[3])});
        put16<STREAM>(p + 4, u32x4{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]),
                                   __float_as_uint(f[7])});
    } else {
        put16<STREAM>(p, u32x4{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]),
                               pack2<T>(f[6], f[7])});
    }
}

// x rounded to an e4m3fn code: nearest, ties to even, NaN past 464 as torch's
// conversion has it (464 is halfway from 448 to the first value past the type,
// and goes to 448).
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b, uint32_t old, bool high) {
    return high ? __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, true) : __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, false);
}
__device__ __forceinline__ float e4m3_overflow(float x) {
    return __builtin_fabsf(x) <= 464.f ? x : __builtin_nanf("");
}
__device__ __forceinline__ void store8_e4m3(uint8_t* p, const float* f) {
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = e4m3_overflow(f[i]);
    uint2 w;
    w.x = e4m3_pair(g[2], g[3], e4m3_pair(g[0], g[1], 0u, false), true);
    w.y = e4m3_pair(g[6], g[7], e4m3_pair(g[4], g[5], 0u, false), true);
    *reinterpret_cast<uint2*>(p) = w;
}

// 8 elements to element offset off of a cache of type code.
__device__ __forceinline__ void store8_cache(void* base, int64_t off, int code, const float* f) {
    if (code == SA_BF16) store8<bf16>(static_cast<bf16*>(base) + off, f);
    else if (code == SA_F16) store8<f16>(static_cast<f16*>(base) + off, f);
    else if (code == SA_F32) store8<float>(static_cast<float*>(base) + off, f);
    else store8_e4m3(static_cast<uint8_t*>(base) + off, f);
}

// 1 / sqrt(x), off by 3/4 of a step at most (v_rsq_f32, which takes arguments below
// the normal range for zero: those are scaled, exactly, on both sides of it).
__device__ __forceinline__ float rsqrt_of(float x) {
    const bool small = x < 0x1p-126f;
    const float r = fast_rsqrt(small ? x * 0x1p32f : x);
    return small ? r * 0x1p16f : r;
}

// Sum over the L lanes of a row, in each of them.
template <int L>
__device__ __forceinline__ float row_sum(float v) {
    if constexpr (L >= 2) v += dpp_mov<0xB1>(v);
    if constexpr (L >= 4) v += dpp_mov<0x4E>(v);
    if constexpr (L >= 8) v += dpp_mov<0x141>(v);
    if constexpr (L >= 16) v += dpp_mov<0x140>(v);
    if constexpr (L >= 32) v += __shfl_xor(v, 16);
    return v;
}

// 8 weights from column d (ones without weights).
template <typename T>
__device__ __forceinline__ void load_weight(const void* w, int w32, int d, float* f) {
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 1.f;
    } else if (w32) {
        load8<float>(static_cast<const float*>(w) + d, f);
    } else {
        load8<T>(static_cast<const T*>(w) + d, f);
    }
}

// Where a lane works: its column pair, its token, its first head.
template <int L>
struct Place {
    int c, h, step;  // first column of the low chunk; first head and heads between two of the group's rows
    int token;       // token of the wave's tile
    bool live;       // whether the column lies in the row
    __device__ __forceinline__ Place(const NormParams& p) {
        const int lane = threadIdx.x & 63;
        const int group = lane / L;
        c = (lane % L) * 8;
        live = c < p.D / 2;
        step = 1 << p.logHG;
        h = group & (step - 1);
        token = group >> p.logHG;
    }
};

// Table row of token m.
__device__ __forceinline__ int position_of(const NormParams& p, int b, int t) {
    const int pos = p.pos ? p.pos[b * p.pos_b + t] : t;
    return min(max(pos, 0), p.n_pos - 1);
}

template <typename T, int L, bool SERVE, bool STREAM>
__global__ __launch_bounds__(64 * kBlockWaves) void norm_rope_kernel(NormParams p) {
    const int chunk = blockIdx.y;
    const int si = chunk >= p.first[2] ? 2 : chunk >= p.first[1] ? 1 : 0;
    const NormSide& s = p.side[si];
    const Place<L> at(p);
    const int h0 = (chunk - p.first[si]) * p.CH, h1 = min(s.H, h0 + p.CH);
    const int tile_tokens = (64 / L) >> p.logHG;
    const int wave = blockIdx.x * kBlockWaves + (threadIdx.x >> 6);
    const int half = p.D / 2;
    const float inv_d = 1.f / static_cast<float>(p.D);
    float wl[8], wh[8];
    if (at.live && s.norm) {
        load_weight<T>(s.w, p.w32, at.c, wl);
        load_weight<T>(s.w, p.w32, at.c + half, wh);
    }
    const int m = wave * tile_tokens + at.token;
    if (m >= p.n_tokens) return;  // (whole rows: the lanes of a row leave together)
    const int b = m / p.T, t = m - b * p.T;
    float cv[8], sv[8];
    if (at.live && s.norm) {
        const int64_t row = static_cast<int64_t>(position_of(p, b, t)) * half + at.c;
        load8<float>(p.cos + row, cv);
        load8<float>(p.sin + row, sv);
    }
    int64_t yo = b * s.ys[0] + t * s.ys[2];
    if constexpr (SERVE) {
        if (s.cache >= 0) {
            const int slot = p.slots[m];
            const int page = slot / p.page_size;
            if (slot < 0 || page >= p.n_pages) return;
            yo = page * s.ys[0] + (slot - page * p.page_size) * s.ys[2];
        }
    }
    const T* x = static_cast<const T*>(s.x) + b * s.xs[0] + t * s.xs[2] + at.c;
    for (int h = h0 + at.h; h < h1; h += at.step) {
        float a[8], e[8];
        if (at.live) {
            load8<T, STREAM>(x + h * s.xs[1], a);
            load8<T, STREAM>(x + h * s.xs[1] + half, e);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = e[i] = 0.f;
        }
        float ya[8], ye[8];
        if (!SERVE || s.norm) {
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sq = __builtin_fmaf(a[i], a[i], __builtin_fmaf(e[i], e[i], sq));
            const float r = rsqrt_of(__builtin_fmaf(row_sum<L>(sq), inv_d, p.eps));
            if (at.live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float zl = a[i] * r * wl[i], zh = e[i] * r * wh[i];
                    ya[i] = zl * cv[i] - zh * sv[i];
                    ye[i] = zh * cv[i] + zl * sv[i];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) ya[i] = a[i], ye[i] = e[i];
        }
        if (at.live) {
            const int64_t off = yo + h * s.ys[1] + at.c;
            if (SERVE && s.cache >= 0) {
                store8_cache(s.y, off, s.cache, ya);
                store8_cache(s.y, off + half, s.cache, ye);
            } else {
                store8<T, STREAM>(static_cast<T*>(s.y) + off, ya);
                store8<T, STREAM>(static_cast<T*>(s.y) + off + half, ye);
            }
        }
    }
}

// Backward.  A wave keeps dw of its column pair over all its rows; a block adds
// its waves' in a fixed order into its row of p.partial.  STREAM: the reads only;
// with dq and dk written past the caches as well, [4,32/32,4096,128] takes 149 us
// for 140, fp32 [4,32/32,2048,128] 172 for 162.
template <typename T, int L, bool STREAM>
__global__ __launch_bounds__(64 * kBlockWaves) void norm_rope_bwd_kernel(NormParams p) {
    __shared__ float red[kBlockWaves][16 * L];
    const int chunk = blockIdx.y;
    const int si = chunk >= p.first[1] ? 1 : 0;
    const NormSide& s = p.side[si];
    const Place<L> at(p);
    const int h0 = (chunk - p.first[si]) * p.CH, h1 = min(s.H, h0 + p.CH);
    const int tile_tokens = (64 / L) >> p.logHG;
    const int wv = threadIdx.x >> 6;
    const int half = p.D / 2;
    const float inv_d = 1.f / static_cast<float>(p.D);
    float wl[8], wh[8], dl[8], dh[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wl[i] = wh[i] = dl[i] = dh[i] = 0.f;
    if (at.live) {
        load_weight<T>(s.w, p.w32, at.c, wl);
        load_weight<T>(s.w, p.w32, at.c + half, wh);
    }
    for (int tile = blockIdx.x * kBlockWaves + wv; tile < p.n_tiles; tile += gridDim.x * kBlockWaves) {
        const int m = tile * tile_tokens + at.token;
        if (m < p.n_tokens) {
            const int b = m / p.T, t = m - b * p.T;
            float cv[8], sv[8];
            if (at.live) {
                const int64_t row = static_cast<int64_t>(position_of(p, b, t)) * half + at.c;
                load8<float>(p.cos + row, cv);
                load8<float>(p.sin + row, sv);
            }
            const T* x = static_cast<const T*>(s.x) + b * s.xs[0] + t * s.xs[2] + at.c;
            const T* g = static_cast<const T*>(s.g) + b * s.gs[0] + t * s.gs[2] + at.c;
            T* y = static_cast<T*>(s.y) + b * s.ys[0] + t * s.ys[2] + at.c;
            for (int h = h0 + at.h; h < h1; h += at.step) {
                float a[8], e[8], ga[8], ge[8];
                float sq = 0.f, hx = 0.f;
                if (at.live) {
                    load8<T, STREAM>(x + h * s.xs[1], a);
                    load8<T, STREAM>(x + h * s.xs[1] + half, e);
                    load8<T, STREAM>(g + h * s.gs[1], ga);
                    load8<T, STREAM>(g + h * s.gs[1] + half, ge);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float zl = ga[i] * cv[i] + ge[i] * sv[i], zh = ge[i] * cv[i] - ga[i] * sv[i];
                        sq = __builtin_fmaf(a[i], a[i], __builtin_fmaf(e[i], e[i], sq));
                        ga[i] = zl;
                        ge[i] = zh;
                        hx = __builtin_fmaf(zl * wl[i], a[i], __builtin_fmaf(zh * wh[i], e[i], hx));
                    }
                }
                const float r = rsqrt_of(__builtin_fmaf(row_sum<L>(sq), inv_d, p.eps));
                const float mr = row_sum<L>(hx) * inv_d * r * r;
                if (at.live) {
                    float xa[8], xe[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        dl[i] = __builtin_fmaf(ga[i], a[i] * r, dl[i]);
                        dh[i] = __builtin_fmaf(ge[i], e[i] * r, dh[i]);
                        xa[i] = r * (ga[i] * wl[i] - a[i] * mr);
                        xe[i] = r * (ge[i] * wh[i] - e[i] * mr);
                    }
                    store8<T>(y + h * s.ys[1], xa);
                    store8<T>(y + h * s.ys[1] + half, xe);
                }
            }
        }
    }
    if (p.partial == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int o = L; o < 64; o <<= 1) {
            dl[i] += __shfl_xor(dl[i], o);
            dh[i] += __shfl_xor(dh[i], o);
        }
    }
    const int lane = threadIdx.x & 63;
    if (lane < L) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            red[wv][lane * 8 + i] = dl[i];
            red[wv][8 * L + lane * 8 + i] = dh[i];
        }
    }
    __syncthreads();
    float* out = p.partial + (static_cast<int64_t>(chunk) * gridDim.x + blockIdx.x) * p.D;
    for (int d = threadIdx.x; d < p.D; d += 64 * kBlockWaves) {
        const int src = d < half ? d : 8 * L + d - half;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kBlockWaves; ++w) v += red[w][src];
        out[d] = v;
    }
}

// dw[d] = sum of n partial rows, in a fixed order and in 64 bits (the sums over a
// block's rows are what 32 bits round): 16 columns a block, 16 lanes of rows for
// each (4.8 us for 1366 rows of 128).
struct DwParams {
    const float* partial[2];
    void* out[2];
    int n[2];
    int D, code;
};
__global__ __launch_bounds__(256) void norm_dw_kernel(DwParams p) {
    __shared__ double red[16][17];
    const int col = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int d = blockIdx.x * 16 + col;
    const float* src = p.partial[blockIdx.y] + d;
    const int n = p.n[blockIdx.y];
    double v = 0.0;
#pragma unroll 8
    for (int r = r0; r < n; r += 16) v += static_cast<double>(src[static_cast<int64_t>(r) * p.D]);
    red[r0][col] = v;
    __syncthreads();
    if (r0 != 0) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += red[i][col];
    void* out = p.out[blockIdx.y];
    if (out == nullptr) return;
    const float f = static_cast<float>(v);
    if (p.code == SA_F32) static_cast<float*>(out)[d] = f;
    else if (p.code == SA_BF16) static_cast<bf16*>(out)[d] = static_cast<bf16>(f);
    else static_cast<f16*>(out)[d] = static_cast<f16>(f);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
struct NormGrid {
    int lanes, CH, logHG, chunks, tiles;
    int64_t blocks;
};

int lanes_for(int D) {
    int l = 1;
    while (l * 16 < D) l *= 2;
    return l;
}

// Heads per chunk and the shape of a wave's rows.  heads: the heads of each
// side; heads_inner: whether a token's heads lie next to each other.  A chunk
// is halved while the launch has fewer than 16 waves for each CU.  Forward of
// [2,32/8,1023,128] bf16 with 4, 8, 16 and 32: 11.3, 9.9, 9.3 and 10.4 us where
// tokens are neighbours, 9.5, 9.4, 9.3 and 10.5 where heads are; 700 packed tokens
// 6.5, 6.5, 6.0 and 6.0; long ones the same.  The backward of short launches would
// rather have 8 ([2,32/8,1023,128] 20.8 -> 16.8 us, [4,12/12,1024,64] 16.8 -> 12.8:
// a wave's sums of dw cost as much as a row).
NormGrid plan_norm(const int* heads, int sides, int64_t tokens, int D, bool heads_inner) {
    NormGrid g{};
    g.lanes = lanes_for(D);
    const int rows = 64 / g.lanes;
    int most = 1;
    for (int i = 0; i < sides; ++i) most = std::max(most, heads[i]);
    g.CH = most;
    for (;;) {
        g.logHG = 0;
        if (heads_inner)
            while ((2 << g.logHG) <= rows && g.CH % (2 << g.logHG) == 0) ++g.logHG;
        g.chunks = 0;
        for (int i = 0; i < sides; ++i) g.chunks += (heads[i] + g.CH - 1) / g.CH;
        const int per = rows >> g.logHG;
        const int64_t tiles = (tokens + per - 1) / per;
        g.tiles = static_cast<int>(tiles);
        g.blocks = (tiles + kBlockWaves - 1) / kBlockWaves;
        if (tiles * g.chunks >= kCus * 16 || g.CH <= (1 << g.logHG)) return g;
        g.CH = (g.CH + 1) / 2;
    }
}

template <template <typename, int> class Launch, typename T, typename... A>
int by_lanes(int lanes, A... a) {
    switch (lanes) {
        case 1: return Launch<T, 1>::run(a...);
        case 2: return Launch<T, 2>::run(a...);
        case 4: return Launch<T, 4>::run(a...);
        case 8: return Launch<T, 8>::run(a...);
        case 16: return Launch<T, 16>::run(a...);
        default: return Launch<T, 32>::run(a...);
    }
}
template <template <typename, int> class Launch, typename... A>
int by_type(int dtype, int lanes, A... a) {
    if (dtype == SA_BF16) return by_lanes<Launch, bf16>(lanes, a...);
    if (dtype == SA_F16) return by_lanes<Launch, f16>(lanes, a...);
    return by_lanes<Launch, float>(lanes, a...);
}

template <typename T, int L>
struct LaunchFwd {
    static int run(const NormParams& p, dim3 grid, bool stream, hipStream_t st) {
        if (stream) norm_rope_kernel<T, L, false, true><<<grid, 64 * kBlockWaves, 0, st>>>(p);
        else norm_rope_kernel<T, L, false, false><<<grid, 64 * kBlockWaves, 0, st>>>(p);
        return status_from_launch();
    }
};
template <typename T, int L>
struct LaunchServe {
    static int run(const NormParams& p, dim3 grid, hipStream_t st) {
        norm_rope_kernel<T, L, true, false><<<grid, 64 * kBlockWaves, 0, st>>>(p);
        return status_from_launch();
    }
};
template <typename T, int L>
struct LaunchBwd {
    static int run(const NormParams& p, dim3 grid, bool stream, hipStream_t st) {
        if (stream) norm_rope_bwd_kernel<T, L, true><<<grid, 64 * kBlockWaves, 0, st>>>(p);
        else norm_rope_bwd_kernel<T, L, false><<<grid, 64 * kBlockWaves, 0, st>>>(p);
        return status_from_launch();
    }
};

bool float_type(int t) { return t == SA_F32 || t == SA_F16 || t == SA_BF16; }

// n element strides that are multiples of 16 bytes, the last one 1.
bool strides16(const int64_t* s, int n, int code) {
    const int per = code == SA_F32 ? 4 : code == SA_FP8_E4M3FN ? 16 : 8;
    for (int i = 0; i < n - 1; ++i)
        if (s[i] % per != 0) return false;
    return s[n - 1] == 1;
}

// Sizes and types that every entry point takes (0: go on, 1: nothing to do, < 0: status).
int check_sizes(int B, int Hq, int Hkv, int T, int D, int n_pos, int dtype, int w_dtype) {
    if (B < 0 || T < 0 || Hq < 0 || Hkv < 0 || n_pos < 0) return SA_ERR_BAD_SHAPE;
    if (!float_type(dtype) || (w_dtype != dtype && w_dtype != SA_F32)) return SA_ERR_BAD_DTYPE;
    if (D < 16 || D > 512 || D % 16 != 0) return SA_ERR_UNSUPPORTED;
    const int64_t tokens = static_cast<int64_t>(B) * T;
    // (a launch has fewer than 2^32 threads, at most 128 for each token)
    if (tokens > (int64_t(1) << 24) || Hq > 65535 / 4 || Hkv > 65535 / 4) return SA_ERR_BAD_SHAPE;
    if (tokens == 0 || Hq + Hkv == 0) return 1;
    return n_pos == 0 ? SA_ERR_BAD_SHAPE : 0;
}

NormSide make_side(const void* x, const void* g, void* y, const void* w, const int64_t* xs, const int64_t* gs,
                   const int64_t* ys, int H) {
    NormSide s{};
    s.x = x;
    s.g = g;
    s.y = y;
    s.w = w;
    for (int i = 0; i < 3; ++i) {
        s.xs[i] = xs[i];
        s.gs[i] = gs ? gs[i] : 0;
        s.ys[i] = ys[i];
    }
    s.H = H;
    s.cache = -1;
    s.norm = 1;
    return s;
}

void set_chunks(NormParams& p, const NormGrid& g, const int* heads, int sides) {
    p.CH = g.CH;
    p.logHG = g.logHG;
    p.n_tiles = g.tiles;
    p.first[0] = 0;
    for (int i = 0; i < 3; ++i) p.first[i + 1] = p.first[i] + (i < sides ? (heads[i] + g.CH - 1) / g.CH : 0);
}

// Blocks of the backward's grid along the tokens: about six on each CU in all
// (the partials that they make are added up in 4 us), each with as many tiles as
// the others.  With 3, 6 and 12 (sums of the partials included):
// [4,12/12,1024,64] fp16 13.4, 16.8 and 16.9 us, [2,32/8,1023,128] bf16 16.7, 20.8
// and 20.8, fp32 24.4, 26.1 and 26.1, [4,32/32,4096,128] bf16 138, 140 and 144,
// fp32 [4,32/32,2048,128] 163, 162 and 151.
int64_t bwd_blocks(const NormGrid& g) {
    const int64_t most = std::max<int64_t>(1, kCus * 6 / g.chunks);
    const int64_t rounds = (g.blocks + most - 1) / most;
    return (g.blocks + rounds - 1) / rounds;
}

// Whether a launch over this many rows of D elements goes past the caches: where
// its tensors are larger than the last-level cache (256 MB), lines that nobody
// reads again only push others out.  [4,32/32,4096,128] bf16 forward and
// backward 274 -> 223 us; [2,32/8,1023,128] kernels 31.4 -> 33.9, so smaller
// ones keep to the caches, where the next operator finds their results.  Half
// rows that share a 128-byte line have to keep to them as well, or each line is
// read twice: [12,32/32,1317,96] 273 us streamed, 241 not.
bool streams(int64_t rows, int D, int dtype, int tensors) {
    const int size = dtype == SA_F32 ? 4 : 2;
    return D / 2 * size % 128 == 0 && rows * D * size * tensors > (int64_t(256) << 20);
}

}  // namespace
}  // namespace sa

extern "C" int sa_qk_norm_rope_fwd(const void* q, const void* k, void* q_out, void* k_out, const void* q_weight,
                                   const void* k_weight, const float* cos_table, const float* sin_table,
                                   const int32_t* positions, int64_t pos_stride, int B, int Hq, int Hkv, int T, int D,
                                   int n_pos, const int64_t* q_strides, const int64_t* k_strides,
                                   const int64_t* qo_strides, const int64_t* ko_strides, float eps, int dtype,
                                   int w_dtype, sa_stream_t stream) {
    using namespace sa;
    const int chk = check_sizes(B, Hq, Hkv, T, D, n_pos, dtype, w_dtype);
    if (chk != 0) return chk > 0 ? 0 : chk;
    if ((Hq > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || !k_out)) || !cos_table || !sin_table || !q_strides ||
        !k_strides || !qo_strides || !ko_strides)
        return SA_ERR_NULL_POINTER;
    if (!strides16(q_strides, 4, dtype) || !strides16(k_strides, 4, dtype) || !strides16(qo_strides, 4, dtype) ||
        !strides16(ko_strides, 4, dtype) || !aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) ||
        !aligned16(cos_table) || !aligned16(sin_table) || !aligned16(q_weight) || !aligned16(k_weight))
        return SA_ERR_BAD_STRIDE;
    NormParams p{};
    const int heads[2] = {Hq, Hkv};
    const NormGrid g = plan_norm(heads, 2, static_cast<int64_t>(B) * T, D, q_strides[1] < q_strides[2]);
    p.side[0] = make_side(q, nullptr, q_out, q_weight, q_strides, nullptr, qo_strides, Hq);
    p.side[1] = make_side(k, nullptr, k_out, k_weight, k_strides, nullptr, ko_strides, Hkv);
    set_chunks(p, g, heads, 2);
    p.cos = cos_table;
    p.sin = sin_table;
    p.pos = positions;
    p.pos_b = pos_stride;
    p.eps = eps;
    p.T = T;
    p.D = D;
    p.n_pos = n_pos;
    p.n_tokens = B * T;
    p.w32 = w_dtype == SA_F32;
    const dim3 grid(static_cast<unsigned>(g.blocks), static_cast<unsigned>(g.chunks));
    const bool past = streams(static_cast<int64_t>(B) * T * (Hq + Hkv), D, dtype, 2);
    return by_type<LaunchFwd>(dtype, g.lanes, p, grid, past, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t sa_qk_norm_rope_bwd_workspace_size(int B, int Hq, int Hkv, int T, int D) {
    using namespace sa;
    if (check_sizes(B, Hq, Hkv, T, D, 1, SA_F32, SA_F32) != 0) return 0;
    const int heads[2] = {Hq, Hkv};
    int64_t rows = 0;
    for (int inner = 0; inner < 2; ++inner) {
        const NormGrid g = plan_norm(heads, 2, static_cast<int64_t>(B) * T, D, inner != 0);
        rows = std::max<int64_t>(rows, bwd_blocks(g) * g.chunks);
    }
    return rows * D * 4;
}

extern "C" int sa_qk_norm_rope_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, void* dq,
                                   void* dk, void* dq_weight, void* dk_weight, const void* q_weight,
                                   const void* k_weight, const float* cos_table, const float* sin_table,
                                   const int32_t* positions, int64_t pos_stride, int B, int Hq, int Hkv, int T, int D,
                                   int n_pos, const int64_t* q_strides, const int64_t* k_strides,
                                   const int64_t* dqo_strides, const int64_t* dko_strides, const int64_t* dq_strides,
                                   const int64_t* dk_strides, float eps, int dtype, int w_dtype, float* workspace,
                                   int64_t workspace_bytes, sa_stream_t stream) {
    using namespace sa;
    const int chk = check_sizes(B, Hq, Hkv, T, D, n_pos, dtype, w_dtype);
    if (chk < 0) return chk;
    if (chk > 0) return dq_weight || dk_weight ? SA_ERR_UNSUPPORTED : 0;  // (no row: the caller clears dw)
    if ((Hq > 0 && (!q || !dq_out || !dq)) || (Hkv > 0 && (!k || !dk_out || !dk)) || !cos_table || !sin_table ||
        !q_strides || !k_strides || !dqo_strides || !dko_strides || !dq_strides || !dk_strides)
        return SA_ERR_NULL_POINTER;
    if (!strides16(q_strides, 4, dtype) || !strides16(k_strides, 4, dtype) || !strides16(dqo_strides, 4, dtype) ||
        !strides16(dko_strides, 4, dtype) || !strides16(dq_strides, 4, dtype) || !strides16(dk_strides, 4, dtype) ||
        !aligned16(q) || !aligned16(k) || !aligned16(dq_out) || !aligned16(dk_out) || !aligned16(dq) ||
        !aligned16(dk) || !aligned16(cos_table) || !aligned16(sin_table) || !aligned16(q_weight) ||
        !aligned16(k_weight))
        return SA_ERR_BAD_STRIDE;
    const bool dw = dq_weight || dk_weight;
    if (dw && (!workspace || workspace_bytes < sa_qk_norm_rope_bwd_workspace_size(B, Hq, Hkv, T, D)))
        return SA_ERR_WORKSPACE;
    NormParams p{};
    const int heads[2] = {Hq, Hkv};
    const NormGrid g = plan_norm(heads, 2, static_cast<int64_t>(B) * T, D, q_strides[1] < q_strides[2]);
    p.side[0] = make_side(q, dq_out, dq, q_weight, q_strides, dqo_strides, dq_strides, Hq);
    p.side[1] = make_side(k, dk_out, dk, k_weight, k_strides, dko_strides, dk_strides, Hkv);
    set_chunks(p, g, heads, 2);
    p.cos = cos_table;
    p.sin = sin_table;
    p.pos = positions;
    p.pos_b = pos_stride;
    p.partial = dw ? workspace : nullptr;
    p.eps = eps;
    p.T = T;
    p.D = D;
    p.n_pos = n_pos;
    p.n_tokens = B * T;
    p.w32 = w_dtype == SA_F32;
    const int64_t blocks = bwd_blocks(g);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(g.chunks));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool past = streams(static_cast<int64_t>(B) * T * (Hq + Hkv), D, dtype, 3);
    const int status = by_type<LaunchBwd>(dtype, g.lanes, p, grid, past, st);
    if (status != 0 || !dw) return status;
    DwParams d{};
    d.partial[0] = workspace;
    d.partial[1] = workspace + p.first[1] * blocks * D;
    d.out[0] = dq_weight;
    d.out[1] = dk_weight;
    d.n[0] = static_cast<int>(p.first[1] * blocks);
    d.n[1] = static_cast<int>((p.first[2] - p.first[1]) * blocks);
    d.D = D;
    d.code = w_dtype;
    norm_dw_kernel<<<dim3(static_cast<unsigned>(D / 16), 2), 256, 0, st>>>(d);
    return status_from_launch();
}

extern "C" int sa_paged_qk_norm_rope_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                                            void* v_cache, const void* q_weight, const void* k_weight,
                                            const float* cos_table, const float* sin_table, const int32_t* positions,
                                            const int32_t* slots, int n_tokens, int Hq, int Hkv, int D, int n_pos,
                                            int page_size, int n_pages, const int64_t* q_strides,
                                            const int64_t* k_strides, const int64_t* v_strides,
                                            const int64_t* qo_strides, const int64_t* kc_strides,
                                            const int64_t* vc_strides, float eps, int dtype, int w_dtype,
                                            int cache_dtype, sa_stream_t stream) {
    using namespace sa;
    const int chk = check_sizes(1, Hq, Hkv, n_tokens, D, n_pos, dtype, w_dtype);
    if (chk != 0) return chk > 0 ? 0 : chk;
    if (page_size <= 0 || n_pages < 0 || static_cast<int64_t>(page_size) * n_pages > INT32_MAX) return SA_ERR_BAD_SHAPE;
    if (!float_type(cache_dtype) && cache_dtype != SA_FP8_E4M3FN) return SA_ERR_BAD_DTYPE;
    // (a cache of no pages stores nothing)
    if ((Hq > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || !v || (n_pages > 0 && (!k_cache || !v_cache)))) || !cos_table ||
        !sin_table || !positions || !slots || !q_strides || !k_strides || !v_strides || !qo_strides || !kc_strides || !vc_strides)
        return SA_ERR_NULL_POINTER;
    if (!strides16(q_strides, 3, dtype) || !strides16(k_strides, 3, dtype) || !strides16(v_strides, 3, dtype) ||
        !strides16(qo_strides, 3, dtype) || !strides16(kc_strides, 4, cache_dtype) ||
        !strides16(vc_strides, 4, cache_dtype) || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
        !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(cos_table) ||
        !aligned16(sin_table) || !aligned16(q_weight) || !aligned16(k_weight))
        return SA_ERR_BAD_STRIDE;
    NormParams p{};
    const int heads[3] = {Hq, Hkv, Hkv};
    const NormGrid g = plan_norm(heads, 3, n_tokens, D, q_strides[1] < q_strides[0]);
    const auto packed = [](const int64_t* s, int64_t* out) { out[0] = 0, out[1] = s[1], out[2] = s[0]; };
    int64_t qs[3], ks[3], vs[3], qo[3];
    packed(q_strides, qs);
    packed(k_strides, ks);
    packed(v_strides, vs);
    packed(qo_strides, qo);
    p.side[0] = make_side(q, nullptr, q_out, q_weight, qs, nullptr, qo, Hq);
    p.side[1] = make_side(k, nullptr, k_cache, k_weight, ks, nullptr, kc_strides, Hkv);
    p.side[2] = make_side(v, nullptr, v_cache, nullptr, vs, nullptr, vc_strides, Hkv);
    p.side[1].cache = p.side[2].cache = cache_dtype;
    p.side[2].norm = 0;
    set_chunks(p, g, heads, 3);
    p.cos = cos_table;
    p.sin = sin_table;
    p.pos = positions;
    p.pos_b = 0;
    p.slots = slots;
    p.eps = eps;
    p.T = n_tokens;
    p.D = D;
    p.n_pos = n_pos;
    p.n_tokens = n_tokens;
    p.w32 = w_dtype == SA_F32;
    p.page_size = page_size;
    p.n_pages = n_pages;
    const dim3 grid(static_cast<unsigned>(g.blocks), static_cast<unsigned>(g.chunks));
    return by_type<LaunchServe>(dtype, g.lanes, p, grid, reinterpret_cast<hipStream_t>(stream));
}
