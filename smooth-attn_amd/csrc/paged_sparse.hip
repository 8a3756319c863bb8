// Paged single-token squareplus attention over chosen pages: the bounds of a
// page's keys, the choice of pages by them, and the attention over the chosen.
//
// For a page, min_d and max_d are the smallest and largest value of key column
// d over the page's tokens.  For any key of the page, q_d k_d <= max(q_d min_d,
// q_d max_d), so with Q+ = sum over the G query heads of a KV head of
// max(q, 0) and Q- of min(q, 0),
//   score = sum_d Q+_d max_d + Q-_d min_d
// is at least the group's sum of q . k for every key of the page, and the
// squareplus weight grows with q . k.  Folding the group into two vectors first
// makes the score one product of 2 D terms whatever G is.
//
// Scores are summed in 64 bits.  The products of 16-bit or 8-bit values are
// exact there and their sums all but, so which pages are chosen does not hang
// on the order of the sum: two scores that differ at all in exact arithmetic
// almost never change places, where 32-bit sums would swap pages at the border
// of the choice, and with them a page's whole part of the output.
#include "paged_kernel.hpp"

namespace sa {
namespace {

// One 16-byte chunk of E as floats (exact).
template <typename E>
struct Chunk {
    static constexpr int N = 16 / sizeof(E);
    float f[N];
};
template <typename E>
__device__ __forceinline__ Chunk<E> widen(u32x4 w) {
    Chunk<E> c;
    if constexpr (std::is_same_v<E, fp8e4>) {
        u32x4 lo, hi;
        widen_e4m3x16<bf16>(w, lo, hi);
        const uint32_t ww[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) c.f[i] = elem<bf16>(ww, i);
    } else {
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < Chunk<E>::N; ++i) c.f[i] = elem<E>(ww, i);
    }
    return c;
}
// The floats of a chunk, each a value of E, as E again (exact).
template <typename E>
__device__ __forceinline__ u32x4 narrow(const Chunk<E>& c) {
    uint32_t w[4];
    if constexpr (std::is_same_v<E, fp8e4>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v = __builtin_amdgcn_cvt_pk_fp8_f32(c.f[4 * i], c.f[4 * i + 1], 0u, false);
            w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(c.f[4 * i + 2], c.f[4 * i + 3], v, true);
        }
    } else {
        pack_row16<E>(c.f, w);
    }
    return u32x4{w[0], w[1], w[2], w[3]};
}

// The smaller and the larger value; NaN where either is.
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// ---------------------------------------------------------------------------
// Bounds of the pages that hold tokens [from_b, to_b) of each sequence.
// ---------------------------------------------------------------------------
struct BoundsParams {
    const void* k;
    void* bounds;  // [n_pages][Hkv][2][D]
    const int32_t* table;
    const int32_t* from;
    const int32_t* to;
    int64_t ks[3];  // page, head, row
    int64_t bt_stride;
    int B, Hkv, D, P, logP, max_pages, n_pages;
    int splits;  // waves that share a (sequence, KV head)
    int lpr;     // lanes per row: a power of two
};

// A wave takes every splits-th page of its (sequence, KV head): lpr lanes cover
// a row (or 64 chunks of it at a time), 64 / lpr rows are read at once.
template <typename E>
__global__ __launch_bounds__(256) void paged_bounds_kernel(BoundsParams p) {
    constexpr int N = Chunk<E>::N;
    const int lane = threadIdx.x & 63;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= static_cast<int64_t>(p.B) * p.Hkv * p.splits) return;
    const int part = static_cast<int>(unit % p.splits);
    const int bh = static_cast<int>(unit / p.splits);
    const int b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int to = min(max(p.to[b], 0), p.max_pages << p.logP);
    const int from = max(p.from[b], 0);
    const int chunks = p.D / N;
    const int row0 = lane / p.lpr, rows = 64 / p.lpr;
    const float inf = __builtin_inff();
    for (int j = (from >> p.logP) + part; (static_cast<int64_t>(j) << p.logP) < to; j += p.splits) {
        const int page = p.table[b * p.bt_stride + j];
        if (page < 0 || page >= p.n_pages) continue;
        const int n = min(to - (j << p.logP), p.P);
        const E* src = static_cast<const E*>(p.k) + page * p.ks[0] + h * p.ks[1];
        E* dst = static_cast<E*>(p.bounds) + (static_cast<int64_t>(page) * p.Hkv + h) * 2 * p.D;
        for (int c0 = 0; c0 < chunks; c0 += p.lpr) {
            const int c = c0 + (lane & (p.lpr - 1));
            Chunk<E> lo, hi;
#pragma unroll
            for (int i = 0; i < N; ++i) lo.f[i] = inf, hi.f[i] = -inf;
            if (c < chunks) {
#pragma unroll 4
                for (int r = row0; r < n; r += rows) {
                    const Chunk<E> x = widen<E>(*reinterpret_cast<const u32x4*>(src + r * p.ks[2] + c * N));
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        lo.f[i] = min_nan(lo.f[i], x.f[i]);
                        hi.f[i] = max_nan(hi.f[i], x.f[i]);
                    }
                }
            }
            for (int o = p.lpr; o < 64; o <<= 1) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    lo.f[i] = min_nan(lo.f[i], __shfl_xor(lo.f[i], o));
                    hi.f[i] = max_nan(hi.f[i], __shfl_xor(hi.f[i], o));
                }
            }
            if (row0 == 0 && c < chunks) {
                *reinterpret_cast<u32x4*>(dst + c * N) = narrow<E>(lo);
                *reinterpret_cast<u32x4*>(dst + p.D + c * N) = narrow<E>(hi);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Choice of pages.
// ---------------------------------------------------------------------------
struct SelectParams {
    const void* q;
    const void* bounds;
    const int32_t* table;
    const int32_t* ctx;
    int32_t* pages;  // [B][Hkv][K]
    double* scores;  // [B][Hkv][max_pages]
    int64_t qs0, qs1;
    int64_t bt_stride;
    int B, Hq, Hkv, G, D, P, logP, max_pages, n_pages, K, n_first, n_last;
    int splits;  // waves that share the pages of a (sequence, KV head)
    int lpp;     // lanes per page: a power of two
};

__device__ __forceinline__ int pages_of(const SelectParams& p, int b) {
    const int ctx = min(max(p.ctx[b], 0), p.max_pages << p.logP);
    return (ctx + p.P - 1) >> p.logP;
}

// Scores.  lpp lanes hold a page's 2 D bounds, NCH chunks each (the minima's
// chunks first); the lane's parts of Q- or Q+ stay in registers, in 64 bits.
template <typename QE, typename E, int NCH>
__global__ __launch_bounds__(256) void paged_score_kernel(SelectParams p) {
    constexpr int N = Chunk<E>::N;
    const int lane = threadIdx.x & 63;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= static_cast<int64_t>(p.B) * p.Hkv * p.splits) return;
    const int part = static_cast<int>(unit % p.splits);
    const int bh = static_cast<int>(unit / p.splits);
    const int b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int np = pages_of(p, b);
    if (np <= p.K) return;  // all of them are taken
    const int chunks = p.D / N;
    const int sub = lane & (p.lpp - 1);
    double qv[NCH][N];
    int off[NCH];
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
        const int c = sub + u * p.lpp;
        off[u] = c < 2 * chunks ? c * N : -1;
#pragma unroll
        for (int i = 0; i < N; ++i) qv[u][i] = 0.0;
        if (c >= 2 * chunks) continue;
        const bool upper = c >= chunks;
        const int d0 = (upper ? c - chunks : c) * N;
        for (int g = 0; g < p.G; ++g) {
            const QE* row = static_cast<const QE*>(p.q) + b * p.qs0 + (h * p.G + g) * p.qs1 + d0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = to_f32(row[i]);
                // (NaN stays in both)
                qv[u][i] += upper ? (x < 0.f ? 0.f : x) : (x > 0.f ? 0.f : x);
            }
        }
    }
    const int per = 64 / p.lpp;  // pages at a time
    const int32_t* trow = p.table + b * p.bt_stride;
    const E* base = static_cast<const E*>(p.bounds) + static_cast<int64_t>(h) * 2 * p.D;
    double* out = p.scores + static_cast<int64_t>(bh) * p.max_pages;
    for (int j0 = part * per; j0 < np; j0 += p.splits * per) {
        const int j = j0 + lane / p.lpp;
        const int page = j < np ? min(max(trow[j], 0), p.n_pages - 1) : -1;
        double s = 0.0;
        if (page >= 0) {
            const E* src = base + static_cast<int64_t>(page) * p.Hkv * 2 * p.D;
#pragma unroll
            for (int u = 0; u < NCH; ++u) {
                if (off[u] < 0) continue;
                const Chunk<E> x = widen<E>(*reinterpret_cast<const u32x4*>(src + off[u]));
#pragma unroll
                for (int i = 0; i < N; ++i) s = __builtin_fma(qv[u][i], static_cast<double>(x.f[i]), s);
            }
        }
        for (int o = 1; o < p.lpp; o <<= 1) s += __shfl_xor(s, o);
        if (page >= 0 && sub == 0) out[j] = s;
    }
}

// A score as an integer of the same order (NaN above all).
__device__ __forceinline__ uint64_t order_key(double s) {
    if (!(s == s)) return ~0ull;
    const uint64_t u = __builtin_bit_cast(uint64_t, s == 0.0 ? 0.0 : s);
    return (u >> 63) ? ~u : u | (1ull << 63);
}

constexpr int kPick = 512;   // threads of a choice
constexpr int kBins = 2048;

// Block sums of two counts in one word each (both below 2^31).
struct Scan {
    uint64_t before, total;
};
__device__ __forceinline__ Scan block_scan(uint64_t v, uint64_t* part) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    uint64_t x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t u = __shfl_up(x, off);
        if (lane >= off) x += u;
    }
    __syncthreads();
    if (lane == 63) part[wv] = x;
    __syncthreads();
    Scan s{x - v, 0};
#pragma unroll
    for (int i = 0; i < kPick / 64; ++i) {
        if (i < wv) s.before += part[i];
        s.total += part[i];
    }
    return s;
}

// The pages of one (sequence, KV head): the first n_first, the last n_last and
// the others with the largest scores, ascending.  The border score is found by
// narrowing the range of keys that holds it, by a factor of up to kBins a pass:
// a histogram of the range, and the bin in which the count from above reaches
// what is needed.  Of equal scores at the border the lower pages are taken.
__global__ __launch_bounds__(kPick) void paged_pick_kernel(SelectParams p) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint64_t part[kPick / 64];
    __shared__ uint64_t range[2];
    __shared__ uint32_t found[2];
    const int bh = blockIdx.x, tid = threadIdx.x;
    const int b = bh / p.Hkv;
    const int np = pages_of(p, b);
    int32_t* out = p.pages + static_cast<int64_t>(bh) * p.K;
    if (np <= p.K) {
        for (int i = tid; i < p.K; i += kPick) out[i] = i < np ? i : -1;
        return;
    }
    const double* scores = p.scores + static_cast<int64_t>(bh) * p.max_pages;
    const int first = p.n_first, last = np - p.n_last;  // (n_first + n_last <= K < np)
    uint32_t need = p.K - p.n_first - p.n_last;
    uint64_t border = ~0ull;
    uint32_t ties = 0;  // pages at the border to take
    if (need > 0) {
        // smallest and largest key
        uint64_t lo = ~0ull, hi = 0;
        for (int j = first + tid; j < last; j += kPick) {
            const uint64_t k = order_key(scores[j]);
            lo = smaller(lo, k);
            hi = larger(hi, k);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            lo = smaller<uint64_t>(lo, __shfl_xor(lo, o));
            hi = larger<uint64_t>(hi, __shfl_xor(hi, o));
        }
        if (tid == 0) range[0] = ~0ull, range[1] = 0;
        __syncthreads();
        if ((tid & 63) == 0) {
            atomicMin(reinterpret_cast<unsigned long long*>(&range[0]), lo);
            atomicMax(reinterpret_cast<unsigned long long*>(&range[1]), hi);
        }
        __syncthreads();
        lo = range[0];
        hi = range[1];
        for (;;) {
            const uint64_t width = hi - lo;
            if (width == 0) {
                border = lo;
                ties = need;
                break;
            }
            const int shift = max(0, 64 - static_cast<int>(__builtin_clzll(width)) - 11);
            for (int i = tid; i < kBins; i += kPick) hist[i] = 0;
            __syncthreads();
            for (int j = first + tid; j < last; j += kPick) {
                const uint64_t k = order_key(scores[j]);
                if (k >= lo && k <= hi) atomicAdd(&hist[(k - lo) >> shift], 1u);
            }
            __syncthreads();
            // thread t: the kBins / kPick bins below those of thread t - 1, from the top
            constexpr int kPer = kBins / kPick;
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) mine += hist[kBins - 1 - (tid * kPer + i)];
            const Scan s = block_scan(mine, part);
            if (s.before < need && s.before + mine >= need) {
                uint32_t above = static_cast<uint32_t>(s.before);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const uint32_t n = hist[kBins - 1 - (tid * kPer + i)];
                    if (above < need && above + n >= need) {
                        found[0] = kBins - 1 - (tid * kPer + i);
                        found[1] = need - above;
                        above = need;  // (no later bin)
                    } else if (above < need) {
                        above += n;
                    }
                }
            }
            __syncthreads();
            const uint32_t bin = found[0];
            need = found[1];
            const uint64_t start = lo + (static_cast<uint64_t>(bin) << shift);
            const bool whole = hist[bin] == need;
            __syncthreads();
            if (whole) {  // all keys from here up
                border = start - 1;
                break;
            }
            hi = start + smaller<uint64_t>(hi - start, (1ull << shift) - 1);  // (no sum past 64 bits)
            lo = start;
        }
    }
    // In the order of the pages: those above the border, and of those at it the first ones.
    uint64_t carry = 0;  // taken pages (low half), pages at the border (high half)
    for (int j0 = 0; j0 < np; j0 += kPick) {
        const int j = j0 + tid;
        bool take = false, tie = false;
        if (j < np) {
            const bool always = j < first || j >= last;
            const uint64_t k = always ? 0 : order_key(scores[j]);
            take = always || (border != ~0ull && k > border);
            tie = !always && ties > 0 && k == border;
        }
        Scan s = block_scan((tie ? 1ull << 32 : 0) | (take ? 1 : 0), part);
        s.before += carry;
        const uint32_t tied_before = static_cast<uint32_t>(s.before >> 32);
        const uint32_t at = static_cast<uint32_t>(s.before) + min(tied_before, ties);
        if (take || (tie && tied_before < ties)) out[at] = j;
        carry += s.total;
    }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
int log2_of(int x) { return __builtin_ctz(static_cast<unsigned>(x)); }
int pow2_up(int x) {
    int p = 1;
    while (p < x) p *= 2;
    return p;
}

bool cache_type(int t) { return t == SA_F32 || t == SA_F16 || t == SA_BF16 || t == SA_FP8_E4M3FN; }
int bytes_of(int t) { return t == SA_F32 ? 4 : t == SA_FP8_E4M3FN ? 1 : 2; }

int check_pages(int B, int Hkv, int D, int page_size, int max_pages, int n_pages, int64_t bt_stride, int cache) {
    if (B < 0 || Hkv <= 0 || max_pages < 0 || n_pages < 0) return SA_ERR_BAD_SHAPE;
    if (page_size <= 0 || (page_size & (page_size - 1)) != 0 || page_size > (1 << 20)) return SA_ERR_UNSUPPORTED;
    if (!cache_type(cache)) return SA_ERR_BAD_DTYPE;
    if (D < 8 || D > 1024 || D % 8 != 0 || (cache == SA_FP8_E4M3FN && D % 16 != 0)) return SA_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(max_pages) * page_size > INT32_MAX / 2 ||
        static_cast<int64_t>(B) * Hkv > INT32_MAX / 64)
        return SA_ERR_UNSUPPORTED;
    return bt_stride < max_pages ? SA_ERR_BAD_STRIDE : 0;
}

// Waves for each of `units`: as many as fill 16 waves a CU, at most `most`.
int splits_for(int64_t units, int64_t most) {
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, (256 * 16 + units - 1) / units)));
}

template <typename QE, typename E>
int launch_scores(const SelectParams& p, int nch, unsigned blocks, hipStream_t st) {
    switch (nch) {
        case 1: paged_score_kernel<QE, E, 1><<<blocks, 256, 0, st>>>(p); break;
        case 2: paged_score_kernel<QE, E, 2><<<blocks, 256, 0, st>>>(p); break;
        case 4: paged_score_kernel<QE, E, 4><<<blocks, 256, 0, st>>>(p); break;
        default: paged_score_kernel<QE, E, 8><<<blocks, 256, 0, st>>>(p); break;
    }
    return status_from_launch();
}
template <typename QE>
int launch_scores(const SelectParams& p, int cache, int nch, unsigned blocks, hipStream_t st) {
    if (cache == SA_BF16) return launch_scores<QE, bf16>(p, nch, blocks, st);
    if (cache == SA_F16) return launch_scores<QE, f16>(p, nch, blocks, st);
    if (cache == SA_F32) return launch_scores<QE, float>(p, nch, blocks, st);
    return launch_scores<QE, fp8e4>(p, nch, blocks, st);
}

// Listed tiles per wave at least: 16 (few partials) where the lists fill the
// device, down to one.
int sparse_per(int B, int Hkv, int n_list, int page_size) {
    return split_for(static_cast<int64_t>(B) * Hkv, n_list, page_size);
}

}  // namespace
}  // namespace sa

extern "C" int sa_paged_key_bounds(const void* k_cache, void* bounds, const int32_t* block_table,
                                   const int32_t* from_lens, const int32_t* to_lens, int B, int Hkv, int D,
                                   int page_size, int max_pages, int n_pages, const int64_t* kc_strides,
                                   int64_t bt_stride, int cache_dtype, sa_stream_t stream) {
    using namespace sa;
    const int chk = check_pages(B, Hkv, D, page_size, max_pages, n_pages, bt_stride, cache_dtype);
    if (chk != 0) return chk;
    if (B == 0 || max_pages == 0 || n_pages == 0) return 0;
    if (!k_cache || !bounds || !block_table || !from_lens || !to_lens || !kc_strides) return SA_ERR_NULL_POINTER;
    const int n = 16 / bytes_of(cache_dtype);
    if (kc_strides[3] != 1 || kc_strides[0] % n != 0 || kc_strides[1] % n != 0 || kc_strides[2] % n != 0 ||
        !aligned16(k_cache) || !aligned16(bounds) || D % n != 0)
        return SA_ERR_BAD_STRIDE;
    BoundsParams p{};
    p.k = k_cache;
    p.bounds = bounds;
    p.table = block_table;
    p.from = from_lens;
    p.to = to_lens;
    for (int i = 0; i < 3; ++i) p.ks[i] = kc_strides[i];
    p.bt_stride = bt_stride;
    p.B = B;
    p.Hkv = Hkv;
    p.D = D;
    p.P = page_size;
    p.logP = log2_of(page_size);
    p.max_pages = max_pages;
    p.n_pages = n_pages;
    p.lpr = std::min(64, pow2_up(D / n));
    p.splits = splits_for(static_cast<int64_t>(B) * Hkv, max_pages);
    const int64_t units = static_cast<int64_t>(B) * Hkv * p.splits;
    const unsigned blocks = static_cast<unsigned>((units + 3) / 4);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (cache_dtype == SA_BF16) paged_bounds_kernel<bf16><<<blocks, 256, 0, st>>>(p);
    else if (cache_dtype == SA_F16) paged_bounds_kernel<f16><<<blocks, 256, 0, st>>>(p);
    else if (cache_dtype == SA_F32) paged_bounds_kernel<float><<<blocks, 256, 0, st>>>(p);
    else paged_bounds_kernel<fp8e4><<<blocks, 256, 0, st>>>(p);
    return status_from_launch();
}

extern "C" int64_t sa_paged_select_workspace_size(int B, int Hkv, int max_pages) {
    if (B <= 0 || Hkv <= 0 || max_pages <= 0) return 0;
    return static_cast<int64_t>(B) * Hkv * max_pages * 8;
}

extern "C" int sa_paged_select_pages(const void* q, const void* bounds, const int32_t* block_table,
                                     const int32_t* context_lens, int32_t* pages, int B, int Hq, int Hkv, int D,
                                     int page_size, int max_pages, int n_pages, int top_k, int n_first, int n_last,
                                     const int64_t* q_strides, int64_t bt_stride, int dtype, int cache_dtype,
                                     void* workspace, int64_t workspace_bytes, sa_stream_t stream) {
    using namespace sa;
    const int chk = check_pages(B, Hkv, D, page_size, max_pages, n_pages, bt_stride, cache_dtype);
    if (chk != 0) return chk;
    if (Hq <= 0 || Hq % Hkv != 0 || top_k < 0 || n_first < 0 || n_last < 0 ||
        static_cast<int64_t>(n_first) + n_last > top_k)
        return SA_ERR_BAD_SHAPE;
    if (dtype != SA_F32 && dtype != SA_F16 && dtype != SA_BF16) return SA_ERR_BAD_DTYPE;
    if (B == 0 || top_k == 0) return 0;
    if (!q || !pages || !q_strides || !context_lens || (max_pages > 0 && (!bounds || !block_table)))
        return SA_ERR_NULL_POINTER;
    if (q_strides[3] != 1 || !aligned16(bounds) || D % (16 / bytes_of(cache_dtype)) != 0) return SA_ERR_BAD_STRIDE;
    const bool choose = top_k < max_pages && n_pages > 0;
    if (choose && (!workspace || workspace_bytes < sa_paged_select_workspace_size(B, Hkv, max_pages)))
        return SA_ERR_WORKSPACE;
    SelectParams p{};
    p.q = q;
    p.bounds = bounds;
    p.table = block_table;
    p.ctx = context_lens;
    p.pages = pages;
    p.scores = static_cast<double*>(workspace);
    p.qs0 = q_strides[0];
    p.qs1 = q_strides[1];
    p.bt_stride = bt_stride;
    p.B = B;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.D = D;
    p.P = page_size;
    p.logP = log2_of(page_size);
    p.max_pages = n_pages == 0 ? 0 : max_pages;
    p.n_pages = n_pages;
    p.K = top_k;
    p.n_first = n_first;
    p.n_last = n_last;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (choose) {
        const int chunks = 2 * D * bytes_of(cache_dtype) / 16;
        p.lpp = std::min(64, pow2_up(chunks));
        const int nch = pow2_up((chunks + p.lpp - 1) / p.lpp);
        p.splits = splits_for(static_cast<int64_t>(B) * Hkv, (max_pages + 64 / p.lpp - 1) / (64 / p.lpp));
        const int64_t units = static_cast<int64_t>(B) * Hkv * p.splits;
        const unsigned blocks = static_cast<unsigned>((units + 3) / 4);
        const int status = dtype == SA_BF16  ? launch_scores<bf16>(p, cache_dtype, nch, blocks, st)
                           : dtype == SA_F16 ? launch_scores<f16>(p, cache_dtype, nch, blocks, st)
                                             : launch_scores<float>(p, cache_dtype, nch, blocks, st);
        if (status != 0) return status;
    }
    paged_pick_kernel<<<static_cast<unsigned>(B) * Hkv, kPick, 0, st>>>(p);
    return status_from_launch();
}

extern "C" int64_t sa_paged_sparse_workspace_size(int B, int Hq, int Hkv, int D, int n_listed, int page_size) {
    using namespace sa;
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || n_listed < 0 || page_size <= 0) return 0;
    const int64_t slots = slots_for(n_listed, page_size, sparse_per(B, Hkv, n_listed, page_size));
    return static_cast<int64_t>(B) * Hq * slots * (D + 1) * 4;
}

extern "C" int sa_paged_sparse_decode(const void* q, const void* k_cache, const void* v_cache, void* out,
                                      const int32_t* block_table, const int32_t* context_lens, const int32_t* pages,
                                      int B, int Hq, int Hkv, int D, int page_size, int max_pages, int n_pages,
                                      int n_listed, const int64_t* q_strides, const int64_t* kv_strides,
                                      const int64_t* vv_strides, const int64_t* o_strides, int64_t bt_stride,
                                      float scale, int dtype, float* workspace, int64_t workspace_bytes,
                                      sa_stream_t stream) {
    using namespace sa;
    if (n_listed < 0) return SA_ERR_BAD_SHAPE;
    const int chk = validate_paged(q, k_cache, v_cache, out, block_table, context_lens, B, Hq, Hkv, D, page_size,
                                   max_pages, n_pages, q_strides, kv_strides, vv_strides, o_strides, dtype);
    if (chk != 0) return chk > 0 ? 0 : chk;
    const int64_t listed = static_cast<int64_t>(n_listed) * page_size;
    if (listed > INT32_MAX / 2 || static_cast<int64_t>(B) * Hkv * ((listed + kTile - 1) / kTile) > INT32_MAX / 2)
        return SA_ERR_UNSUPPORTED;
    if (bt_stride < max_pages) return SA_ERR_BAD_STRIDE;
    if (!workspace || (n_listed > 0 && !pages)) return SA_ERR_NULL_POINTER;
    if (workspace_bytes < sa_paged_sparse_workspace_size(B, Hq, Hkv, D, n_listed, page_size)) return SA_ERR_WORKSPACE;
    PagedParams prm{};
    prm.q = q;
    prm.k = k_cache;
    prm.v = v_cache;
    prm.out = static_cast<bf16*>(out);
    prm.table = block_table;
    prm.ctx = context_lens;
    prm.list = pages;
    prm.n_list = n_listed;
    prm.per = sparse_per(B, Hkv, n_listed, page_size);
    prm.n_slots = static_cast<int>(slots_for(n_listed, page_size, prm.per));
    prm.ws_o = workspace;
    prm.ws_s = prm.ws_o + static_cast<int64_t>(B) * Hq * prm.n_slots * D;
    prm.D = D;
    for (int i = 0; i < 4; ++i) {
        prm.qs[i] = q_strides[i];
        prm.ks[i] = kv_strides[i];
        prm.vs[i] = vv_strides[i];
    }
    for (int i = 0; i < 3; ++i) prm.os[i] = o_strides[i];
    prm.bt_stride = bt_stride;
    prm.B = B;
    prm.Hq = Hq;
    prm.Hkv = Hkv;
    prm.G = Hq / Hkv;
    prm.P = page_size;
    prm.logP = log2_of(page_size);
    prm.max_pages = max_pages;
    prm.n_pages = n_pages;
    prm.scale = scale;
    return launch_paged_types<true>(prm, dtype, reinterpret_cast<hipStream_t>(stream));
}
