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

// Two registers with rows exchanged: of lanes that differ in BIT (16 or 32), the
// lower ones get both values of a, the upper ones both of b (r.x from the lower
// lane, r.y from the upper).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int BIT>
__device__ __forceinline__ u32x2 swap_rows(uint32_t a, uint32_t b) {
    if constexpr (BIT == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        return u32x2{r[0], r[1]};
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        return u32x2{r[0], r[1]};
    }
}

// The values of a 16-byte chunk as the bounds compare them: fp32 for fp32 and
// bf16 keys, pairs of fp16 for fp16 and e4m3fn ones (each such value is an fp16
// value), which gfx950 compares two at a time.
template <typename E>
struct Compared {
    static constexpr bool PAIRS = std::is_same_v<E, f16> || std::is_same_v<E, fp8e4>;
    using V = std::conditional_t<PAIRS, f16x2, float>;
    static constexpr int N = PAIRS ? Chunk<E>::N / 2 : Chunk<E>::N;
    // (by value: a cast of an element of a vector takes the first one)
    static __device__ __forceinline__ f16x2 pair(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
    static __device__ __forceinline__ void read(u32x4 w, V* v) {
        if constexpr (std::is_same_v<E, f16>) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = pair(w[i]);
        } else if constexpr (PAIRS) {
            u32x4 lo, hi;
            widen_e4m3x16<f16>(w, lo, hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = pair(lo[i]);
                v[4 + i] = pair(hi[i]);
            }
        } else {
            const Chunk<E> c = widen<E>(w);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = c.f[i];
        }
    }
    static __device__ __forceinline__ u32x4 write(const V* v) {  // (exact)
        if constexpr (std::is_same_v<E, f16>) {
            return u32x4{__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]),
                         __builtin_bit_cast(uint32_t, v[2]), __builtin_bit_cast(uint32_t, v[3])};
        } else {
            Chunk<E> c;
            if constexpr (PAIRS) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    c.f[2 * i] = static_cast<float>(v[i][0]);
                    c.f[2 * i + 1] = static_cast<float>(v[i][1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) c.f[i] = v[i];
            }
            return narrow<E>(c);
        }
    }
    static __device__ __forceinline__ V largest() {
        if constexpr (PAIRS) return __builtin_bit_cast(f16x2, 0x7C007C00u);  // infinity
        else return __builtin_inff();
    }
    static __device__ __forceinline__ V smaller_of(V a, V b) { return __builtin_elementwise_minimum(a, b); }  // (NaN stays)
    template <int CTRL>
    static __device__ __forceinline__ V moved(V v) {
        return __builtin_bit_cast(V, dpp_mov<CTRL>(__builtin_bit_cast(float, v)));
    }
    template <int BIT>
    static __device__ __forceinline__ V over_rows(V a, V b) {
        const u32x2 r = swap_rows<BIT>(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
        return smaller_of(__builtin_bit_cast(V, static_cast<uint32_t>(r.x)), __builtin_bit_cast(V, static_cast<uint32_t>(r.y)));
    }
};

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
};

// A wave takes every splits-th page of its (sequence, KV head): LPR lanes cover a
// row (or 64 chunks of it at a time) and 64 / LPR rows are read at once, kAhead
// such reads before the first is used.  Largest values are kept as smallest
// negated ones, so both are the same operation: at the last exchange the lower
// half of the wave takes over the one kind and the upper half the other.  Four
// prompts of 8192 to 16384 tokens, Hkv 8, D = 128 bf16: 26 us, 4.4 TB/s (37 us with
// both kinds exchanged over LDS and one page's loads behind another's); fp32 keys
// 47 us, 5.2 TB/s.  Where kAhead reads are more rows than a page has, they read and
// compare its last row again: at pages of 16 half of the rows of e4m3fn keys (22 us,
// 2.7 TB/s) and of D = 64 bf16 ones (20 us, 3.0 TB/s), three quarters of D = 64
// e4m3fn ones (22 us, 1.4 TB/s).
constexpr int kAhead = 4;
template <typename E, int LPR>
__global__ __launch_bounds__(256) void paged_bounds_kernel(BoundsParams p) {
    using C = Compared<E>;
    using V = typename C::V;
    constexpr int N = Chunk<E>::N;
    constexpr int ROWS = 64 / LPR;
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= static_cast<uint32_t>(p.B * p.Hkv) * p.splits) return;
    const int bh = unit / static_cast<uint32_t>(p.splits), part = unit - bh * p.splits;
    const int b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int to = min(max(p.to[b], 0), p.max_pages << p.logP);
    const int from = max(p.from[b], 0);
    const int chunks = p.D / N;
    const int row0 = lane / LPR;
    const int32_t* trow = p.table + b * p.bt_stride;
    const int end = (to + p.P - 1) >> p.logP;
    int j = (from >> p.logP) + part;
    int next = j < end ? trow[j] : -1;
    for (; j < end; j += p.splits) {
        const int page = next;
        if (j + p.splits < end) next = trow[j + p.splits];
        if (page < 0 || page >= p.n_pages) continue;
        const int n = min(to - (j << p.logP), p.P);
        const E* src = static_cast<const E*>(p.k) + page * p.ks[0] + h * p.ks[1];
        E* dst = static_cast<E*>(p.bounds) + (static_cast<int64_t>(page) * p.Hkv + h) * 2 * p.D;
        for (int c0 = 0; c0 < chunks; c0 += LPR) {
            const int c = c0 + (lane & (LPR - 1));
            const E* col = src + min(c, chunks - 1) * N;
            V lo[C::N], hi[C::N];  // smallest values, and smallest negated ones
#pragma unroll
            for (int i = 0; i < C::N; ++i) lo[i] = hi[i] = C::largest();
            for (int r0 = 0; r0 < n; r0 += kAhead * ROWS) {
                u32x4 w[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a)  // (a row that is read twice changes nothing)
                    w[a] = load16(col + min(r0 + a * ROWS + row0, n - 1) * p.ks[2]);
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    V x[C::N];
                    C::read(w[a], x);
#pragma unroll
                    for (int i = 0; i < C::N; ++i) {
                        lo[i] = C::smaller_of(lo[i], x[i]);
                        hi[i] = C::smaller_of(hi[i], -x[i]);
                    }
                }
            }
            V out[C::N];
            auto both = [&](int i, auto other) {
                lo[i] = C::smaller_of(lo[i], other(lo[i]));
                hi[i] = C::smaller_of(hi[i], other(hi[i]));
            };
#pragma unroll
            for (int i = 0; i < C::N; ++i) {
                if constexpr (LPR <= 1) both(i, [](V v) { return C::template moved<0xB1>(v); });
                if constexpr (LPR <= 2) both(i, [](V v) { return C::template moved<0x4E>(v); });
                if constexpr (LPR <= 4) both(i, [](V v) { return C::template moved<0x124>(v); });
                if constexpr (LPR <= 8) both(i, [](V v) { return C::template moved<0x128>(v); });
                if constexpr (LPR <= 16) {
                    lo[i] = C::template over_rows<16>(lo[i], lo[i]);
                    hi[i] = C::template over_rows<16>(hi[i], hi[i]);
                }
                if constexpr (LPR <= 32) {
                    out[i] = C::template over_rows<32>(lo[i], hi[i]);
                    if (lane >= 32) out[i] = -out[i];
                } else {
                    out[i] = lo[i];
                }
            }
            if (c >= chunks) continue;
            if constexpr (LPR <= 32) {
                if ((lane & 31) < LPR) *reinterpret_cast<u32x4*>(dst + (lane >= 32 ? p.D : 0) + c * N) = C::write(out);
            } else {
                *reinterpret_cast<u32x4*>(dst + c * N) = C::write(out);
#pragma unroll
                for (int i = 0; i < C::N; ++i) out[i] = -hi[i];
                *reinterpret_cast<u32x4*>(dst + p.D + c * N) = C::write(out);
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
    int qcode;
};

__device__ __forceinline__ int pages_of(const SelectParams& p, int b) {
    const int ctx = min(max(p.ctx[b], 0), p.max_pages << p.logP);
    return (ctx + p.P - 1) >> p.logP;
}

// N query values from column d, in floats (N = 4, 8 or 16; rows of 16-byte multiples).
template <int N>
__device__ __forceinline__ void load_query(const void* row, int code, int d, float* f) {
    if (code == SA_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const float*>(row) + d + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i + j] = __uint_as_float(w[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + d + i);
            const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i + j] = code == SA_BF16 ? elem<bf16>(ww, j) : elem<f16>(ww, j);
        }
    }
}

// The value of the lane that differs from this one in bit BIT of its number
// (4: and in the two below it).
template <int BIT>
__device__ __forceinline__ double from_other(double v) {
    if constexpr (BIT >= 16) {
        return __shfl_xor(v, BIT);
    } else {
        constexpr int ctrl = BIT == 1 ? 0xB1 : BIT == 2 ? 0x4E : BIT == 4 ? 0x141 : 0x128;
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const float lo = dpp_mov<ctrl>(__uint_as_float(static_cast<uint32_t>(u)));
        const float hi = dpp_mov<ctrl>(__uint_as_float(static_cast<uint32_t>(u >> 32)));
        return __builtin_bit_cast(double, static_cast<uint64_t>(__float_as_uint(hi)) << 32 | __float_as_uint(lo));
    }
}

// Sums of COUNT values over groups of 2 BIT lanes.  While a lane has several
// values, each of two partners keeps half of them and takes the other's part, so
// COUNT sums cost about as many exchanges as two whole ones; what is left in v[0
// .. max(1, COUNT / (2 BIT))) belongs to the value that first_value names.
template <int BIT, int COUNT>
__device__ __forceinline__ void group_sums(double* v) {
    if constexpr (COUNT > 1 && BIT >= 16) {
#pragma unroll
        for (int i = 0; i < COUNT / 2; ++i) {
            const uint64_t a = __builtin_bit_cast(uint64_t, v[i]), b = __builtin_bit_cast(uint64_t, v[i + COUNT / 2]);
            const u32x2 lo = swap_rows<BIT>(static_cast<uint32_t>(a), static_cast<uint32_t>(b));
            const u32x2 hi = swap_rows<BIT>(static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b >> 32));
            v[i] = __builtin_bit_cast(double, static_cast<uint64_t>(hi.x) << 32 | lo.x) +
                   __builtin_bit_cast(double, static_cast<uint64_t>(hi.y) << 32 | lo.y);
        }
    } else if constexpr (COUNT > 1) {
        const bool upper = (threadIdx.x & BIT) != 0;
#pragma unroll
        for (int i = 0; i < COUNT / 2; ++i) {
            const double keep = upper ? v[i + COUNT / 2] : v[i];
            const double send = upper ? v[i] : v[i + COUNT / 2];
            v[i] = keep + from_other<BIT>(send);
        }
    } else {
        v[0] += from_other<BIT>(v[0]);
    }
    if constexpr (BIT > 1) group_sums<BIT / 2, COUNT / 2 < 1 ? 1 : COUNT / 2>(v);
}
template <int BIT, int COUNT>
__device__ __forceinline__ int first_value() {
    if constexpr (COUNT > 1 && BIT >= 1) {
        const int mine = (threadIdx.x & BIT) != 0 ? COUNT / 2 : 0;
        return mine + first_value<BIT / 2, COUNT / 2>();
    } else {
        return 0;
    }
}

// Scores.  LPP lanes hold a page's 2 D bounds, NCH chunks each (the minima's
// chunks first); the lane's parts of Q- and Q+ stay in registers, in 64 bits.  A
// wave takes kBatch loads' pages at a time: their table entries are read a batch
// ahead, their bounds all before the first is used, and their sums are added up
// together.  Bound by memory, 512 bytes a page and KV head anywhere in it: 138 MB
// (64 sequences of 512 to 16384 tokens) 35 us, 201 MB (8 of 65536 to 131072) 42;
// with one load in flight and each sum exchanged alone 83 and 88.
constexpr int kBatch = 8;
template <typename E, int LPP, int NCH>
__global__ __launch_bounds__(256) void paged_score_kernel(SelectParams p) {
    constexpr int N = Chunk<E>::N;
    constexpr int PER = 64 / LPP;  // pages of one load
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= static_cast<uint32_t>(p.B * p.Hkv) * p.splits) return;
    const int bh = unit / static_cast<uint32_t>(p.splits), part = unit - bh * p.splits;
    const int b = bh / p.Hkv, h = bh - b * p.Hkv;
    int j0 = part * PER * kBatch;
    const int step = p.splits * PER * kBatch;
    const int chunks = p.D / N;
    const int sub = lane & (LPP - 1), mine = lane / LPP;
    // The length, the table entries and the queries are all read at once: entries
    // past the sequence's pages are read, and not used.
    const int32_t* trow = p.table + b * p.bt_stride;
    const int np = pages_of(p, b);
    int page[kBatch];
    auto read_table = [&](int j) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) page[u] = trow[min(j + u * PER + mine, p.max_pages - 1)];
    };
    read_table(j0);
    double qv[NCH][N];
    int off[NCH];
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
        const int c = sub + u * LPP;
        off[u] = min(c, 2 * chunks - 1) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) qv[u][i] = 0.0;
        if (c >= 2 * chunks) continue;
        const bool upper = c >= chunks;
        const int d0 = (upper ? c - chunks : c) * N;
        for (int g0 = 0; g0 < p.G; g0 += 4) {
            float x[4][N];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int64_t row = b * p.qs0 + (h * p.G + min(g0 + g, p.G - 1)) * p.qs1;
                load_query<N>(static_cast<const char*>(p.q) + row * (p.qcode == SA_F32 ? 4 : 2), p.qcode, d0, x[g]);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (g0 + g >= p.G) continue;
#pragma unroll
                for (int i = 0; i < N; ++i)  // (NaN stays in both)
                    qv[u][i] += upper ? (x[g][i] < 0.f ? 0.f : x[g][i]) : (x[g][i] > 0.f ? 0.f : x[g][i]);
            }
        }
    }
    if (np <= p.K) return;  // all of them are taken
    const int64_t page_size = static_cast<int64_t>(p.Hkv) * 2 * p.D;
    const E* base = static_cast<const E*>(p.bounds) + static_cast<int64_t>(h) * 2 * p.D;
    double* out = p.scores + static_cast<int64_t>(bh) * p.max_pages;
    constexpr int LEFT = kBatch / LPP < 1 ? 1 : kBatch / LPP;  // sums that a lane ends up with
    const int u0 = first_value<LPP / 2, kBatch>();
    for (; j0 < np; j0 += step) {
        u32x4 w[kBatch][NCH];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const E* src = base + min(max(page[u], 0), p.n_pages - 1) * page_size;
#pragma unroll
            for (int c = 0; c < NCH; ++c) w[u][c] = load16(src + off[c]);  // (past the caches: read once)
        }
        if (j0 + step < np) read_table(j0 + step);
        double s[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            s[u] = 0.0;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                if (2 * chunks < LPP * NCH && sub + c * LPP >= 2 * chunks) continue;  // (no such chunk)
                const Chunk<E> x = widen<E>(w[u][c]);
#pragma unroll
                for (int i = 0; i < N; ++i) s[u] = __builtin_fma(qv[c][i], static_cast<double>(x.f[i]), s[u]);
            }
        }
        group_sums<LPP / 2, kBatch>(s);
        // (lanes below the last exchange hold the same sum: the lowest writes it)
        if (LPP <= kBatch || (sub & (LPP / kBatch - 1)) == 0) {
#pragma unroll
            for (int i = 0; i < LEFT; ++i) {
                const int j = j0 + (u0 + i) * PER + mine;
                if (j < np) out[j] = s[i];
            }
        }
    }
}

// A score as an integer of the same order, above 2^32 (NaN above all).
__device__ __forceinline__ uint64_t order_key(double s) {
    const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);  // (-0 becomes 0)
    const uint64_t m = static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | (1ull << 63);
    return s == s ? u ^ m : ~0ull;
}

// Inclusive prefix sum, smallest and largest over the 64 lanes of a wave, by DPP:
// rows of 16 first (row_shr, mirrors), then over the rows.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t old, uint32_t v) {
    return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
    v += dpp_u32<0x111>(0, v);
    v += dpp_u32<0x112>(0, v);
    v += dpp_u32<0x114>(0, v);
    v += dpp_u32<0x118>(0, v);
    v += dpp_u32<0x142, 0xA>(0, v);  // row_bcast:15 into rows 1 and 3
    v += dpp_u32<0x143, 0xC>(0, v);  // row_bcast:31 into rows 2 and 3
    return v;
}
template <typename F>
__device__ __forceinline__ uint32_t wave_all(uint32_t v, F f) {
    v = f(v, dpp_u32<0xB1>(v, v));
    v = f(v, dpp_u32<0x4E>(v, v));
    v = f(v, dpp_u32<0x141>(v, v));
    v = f(v, dpp_u32<0x140>(v, v));
    const auto at = [&](int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, l)); };
    return f(f(at(0), at(16)), f(at(32), at(48)));
}

constexpr int kBins = 2048;
constexpr int kRanked = 256;  // keys that are ranked one against another

// The pages of one (sequence, KV head): the first n_first, the last n_last and
// the others with the largest scores, ascending; of equal scores at the border
// the lower pages.
//
// The border score is found by narrowing the range of keys that holds it: a
// histogram of the range in LDS, and the bin in which the count from above
// reaches what is needed, a factor of up to kBins a pass.  Once at most kRanked
// keys are left they are ranked against each other (one pass, over the keys' high
// halves, and about ten keys for a few thousand scores).  The pages taken are
// bits in LDS, and the sums of their counts place them in order.
//
// A thread keeps its keys in registers, all read at once.  One block's waves
// share a CU, so what bounds this is the instructions for each key: with
// compares of the position and of both ends of the range in 64 bits, and a
// ballot for every 64 pages instead of the bits, 64 lists of up to 8192 pages
// took 13.4 us, and with the keys read from memory in every pass 30.5.  KEYS = 0:
// any number of pages, read in every pass.
template <int THREADS, int KEYS>
__global__ __launch_bounds__(THREADS) void paged_pick_kernel(SelectParams p) {
    constexpr int WAVES = THREADS / 64;
    constexpr int WORDS = KEYS > 0 ? KEYS * THREADS / 32 : 1;
    static_assert(WORDS <= THREADS, "a thread for each word of the bits");
    __shared__ uint32_t hist[kBins];
    __shared__ uint64_t ranked[kRanked];
    __shared__ uint32_t sums[2][WAVES];
    __shared__ uint32_t bits[2][WORDS];  // pages taken, pages at the border
    __shared__ uint32_t found[4];        // bin, needed from it, keys in it; keys ranked so far
    __shared__ uint64_t border_at;
    __shared__ uint32_t ties_at;
    const int bh = blockIdx.x, tid = threadIdx.x;
    const int lane = tid & 63, wv = tid >> 6;
    const int b = bh / p.Hkv;
    const int np = pages_of(p, b);
    int32_t* out = p.pages + static_cast<int64_t>(bh) * p.K;
    const double* scores = p.scores + static_cast<int64_t>(bh) * p.max_pages;
    double v[KEYS > 0 ? KEYS : 1];
    if (KEYS > 0 && p.K < p.max_pages) {  // (else there are no scores; those past the sequence's pages are not used)
#pragma unroll
        for (int i = 0; i < KEYS; ++i) v[i] = scores[min(i * THREADS + tid, p.max_pages - 1)];
    }
    for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
    if (tid < WORDS) bits[0][tid] = bits[1][tid] = 0;
    if (np <= p.K) {
        for (int i = tid; i < p.K; i += THREADS) out[i] = i < np ? i : -1;
        return;
    }
    const int first = p.n_first, last = np - p.n_last;  // (n_first + n_last <= K < np)
    // Keys of the pages that compete, 0 for the others.
    uint64_t mine[KEYS > 0 ? KEYS : 1];
    if constexpr (KEYS > 0) {
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            const int j = i * THREADS + tid;
            mine[i] = j >= first && j < last ? order_key(v[i]) : 0;
        }
    }
    auto each = [&](auto f) {
        if constexpr (KEYS > 0) {
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
                if (i * THREADS < np) f(mine[i], i * THREADS + tid);  // (the same for all threads)
            }
        } else {
            for (int j = first + tid; j < last; j += THREADS) f(order_key(scores[j]), j);
        }
    };
    uint32_t need = p.K - p.n_first - p.n_last;
    uint64_t border = ~0ull;
    uint32_t ties = 0;  // pages at the border to take
    if (need > 0) {
        // The range, from the keys' high halves (0 less 1 is the largest number).
        uint32_t least = ~0u, most = 0;
        each([&](uint64_t k, int) {
            const uint32_t h = static_cast<uint32_t>(k >> 32);
            least = smaller(least, h - 1);
            most = larger(most, h);
        });
        least = wave_all(least, [](uint32_t x, uint32_t y) { return smaller(x, y); });
        most = wave_all(most, [](uint32_t x, uint32_t y) { return larger(x, y); });
        if (lane == 0) sums[0][wv] = least, sums[1][wv] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            least = smaller(least, sums[0][i]);
            most = larger(most, sums[1][i]);
        }
        ++least;
        uint64_t lo = static_cast<uint64_t>(least) << 32, hi = static_cast<uint64_t>(most) << 32 | 0xFFFFFFFFu;
        int shift = 32 + max(0, 32 - static_cast<int>(__builtin_clz(most - least | 1)) - 11);
        each([&](uint64_t k, int) {
            const uint32_t h = static_cast<uint32_t>(k >> 32);
            if (h != 0) atomicAdd(&hist[(h - least) >> (shift - 32)], 1u);
        });
        for (;;) {
            __syncthreads();
            // thread t: the bins below those of thread t - 1, from the top
            constexpr int PER = kBins / THREADS;
            uint32_t count[PER], sum = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                uint32_t& bin = hist[kBins - 1 - (tid * PER + i)];
                sum += count[i] = bin;
                bin = 0;
            }
            const uint32_t upto = wave_upto(sum);
            if (lane == 63) sums[0][wv] = upto;
            if (tid == 0) found[3] = 0;
            __syncthreads();
            uint32_t above = upto - sum;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) above += i < wv ? sums[0][i] : 0u;
            if (above < need && above + sum >= need) {  // (one thread, one of its bins)
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    if (above < need && above + count[i] >= need) {
                        found[0] = kBins - 1 - (tid * PER + i);
                        found[1] = need - above;
                        found[2] = count[i];
                    }
                    above += count[i];
                }
            }
            __syncthreads();
            need = found[1];
            const uint32_t left = found[2];
            lo += static_cast<uint64_t>(found[0]) << shift;
            hi = lo + smaller<uint64_t>(hi - lo, (1ull << shift) - 1);  // (no sum past 64 bits)
            if (left == need) {  // all keys from here up
                border = lo - 1;
                break;
            }
            if (lo == hi) {
                border = lo;
                ties = need;
                break;
            }
            if (left <= kRanked) {
                each([&](uint64_t k, int) {
                    if (k - lo <= hi - lo) ranked[atomicAdd(&found[3], 1u)] = k;
                });
                __syncthreads();
                for (uint32_t r = tid; r < left; r += THREADS) {
                    const uint64_t k = ranked[r];
                    uint32_t over = 0, same = 0;
                    for (uint32_t i = 0; i < left; ++i) {
                        over += ranked[i] > k;
                        same += ranked[i] == k;
                    }
                    if (over < need && over + same >= need) {  // (equal keys say the same)
                        border_at = k;
                        ties_at = need - over;
                    }
                }
                __syncthreads();
                border = border_at;
                ties = ties_at;
                break;
            }
            __syncthreads();  // found has been read
            shift = max(0, 64 - static_cast<int>(__builtin_clzll(hi - lo)) - 11);
            each([&](uint64_t k, int) {
                if (k - lo <= hi - lo) atomicAdd(&hist[(k - lo) >> shift], 1u);
            });
        }
    }
    // Which pages, and where: those above the border, the first of those at it,
    // and the first and last ones.
    if constexpr (KEYS > 0) {
        if (need == 0) __syncthreads();  // (the bits are clear)
        each([&](uint64_t k, int j) {
            if (k > border) atomicOr(&bits[0][j >> 5], 1u << (j & 31));
        });
        if (ties > 0)
            each([&](uint64_t k, int j) {
                if (k == border) atomicOr(&bits[1][j >> 5], 1u << (j & 31));
            });
        for (int i = tid; i < p.n_first + p.n_last; i += THREADS) {
            const int j = i < first ? i : last + i - first;
            atomicOr(&bits[0][j >> 5], 1u << (j & 31));
        }
        __syncthreads();
        // Sum over the words before this thread's.
        auto before = [&](uint32_t n, uint32_t* part) {
            const uint32_t upto = wave_upto(n);
            if (lane == 63) part[wv] = upto;
            __syncthreads();
            uint32_t all = upto - n;
#pragma unroll
            for (int i = 0; i < (WORDS + 63) / 64; ++i) all += i < wv ? part[i] : 0u;
            return all;
        };
        uint32_t word = tid < WORDS ? bits[0][tid] : 0u;
        if (ties > 0) {
            uint32_t tied = tid < WORDS ? bits[1][tid] : 0u;
            const uint32_t done = before(__popc(tied), sums[0]);
            for (uint32_t n = done; n < ties && tied != 0; ++n) {
                word |= tied & (0u - tied);
                tied &= tied - 1;
            }
        }
        uint32_t at = before(__popc(word), sums[1]);
        for (; word != 0; word &= word - 1) out[at++] = tid * 32 + __builtin_ctz(word);
    } else {
        uint32_t before[2] = {0, 0};
        const uint64_t below = (1ull << lane) - 1;
        for (int j0 = 0; j0 < np; j0 += THREADS) {
            const int j = j0 + tid;
            const bool always = j < first || (j >= last && j < np);
            const uint64_t k = !always && j < last ? order_key(scores[j]) : 0;
            const bool take = always || k > border, tie = ties > 0 && k == border;
            const uint64_t takes = __ballot(take), tied = __ballot(tie);
            if (lane == 0) sums[0][wv] = __popcll(takes), sums[1][wv] = __popcll(tied);
            __syncthreads();
            uint32_t at[2] = {before[0], before[1]};
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    at[c] += i < wv ? sums[c][i] : 0u;
                    before[c] += sums[c][i];
                }
            }
            const uint32_t t = at[1] + __popcll(tied & below);
            if (take || (tie && t < ties)) out[at[0] + __popcll(takes & below) + smaller(t, ties)] = j;
            __syncthreads();
        }
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
        static_cast<int64_t>(B) * Hkv > INT32_MAX / 1024)  // (the choice's blocks of up to 1024 threads: below 2^32)
        return SA_ERR_UNSUPPORTED;
    return bt_stride < max_pages ? SA_ERR_BAD_STRIDE : 0;
}

// Waves for each of `units`: as many as fill 16 waves a CU, at most `most`.  With 8,
// 16 and 32: bounds of four prompts 31.7, 25.5 and 25.0 us, after a token of each of
// 64 sequences 2.8, 3.0 and 3.7; scores and choice for those of 512 to 16384 tokens
// 42.5, 36.3 and 37.4, for 8 of 65536 to 131072 50, 49 and 50.
int splits_for(int64_t units, int64_t most) {
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, (256 * 16 + units - 1) / units)));
}

template <typename E>
int launch_bounds(const BoundsParams& p, int lpr, unsigned blocks, hipStream_t st) {
    switch (lpr) {
        case 1: paged_bounds_kernel<E, 1><<<blocks, 256, 0, st>>>(p); break;
        case 2: paged_bounds_kernel<E, 2><<<blocks, 256, 0, st>>>(p); break;
        case 4: paged_bounds_kernel<E, 4><<<blocks, 256, 0, st>>>(p); break;
        case 8: paged_bounds_kernel<E, 8><<<blocks, 256, 0, st>>>(p); break;
        case 16: paged_bounds_kernel<E, 16><<<blocks, 256, 0, st>>>(p); break;
        case 32: paged_bounds_kernel<E, 32><<<blocks, 256, 0, st>>>(p); break;
        default: paged_bounds_kernel<E, 64><<<blocks, 256, 0, st>>>(p); break;
    }
    return status_from_launch();
}

template <typename E>
int launch_scores(const SelectParams& p, int lpp, int nch, unsigned blocks, hipStream_t st) {
    switch (lpp * nch) {
        case 2: paged_score_kernel<E, 2, 1><<<blocks, 256, 0, st>>>(p); break;
        case 4: paged_score_kernel<E, 4, 1><<<blocks, 256, 0, st>>>(p); break;
        case 8: paged_score_kernel<E, 8, 1><<<blocks, 256, 0, st>>>(p); break;
        case 16: paged_score_kernel<E, 16, 1><<<blocks, 256, 0, st>>>(p); break;
        case 32: paged_score_kernel<E, 32, 1><<<blocks, 256, 0, st>>>(p); break;
        case 64: paged_score_kernel<E, 64, 1><<<blocks, 256, 0, st>>>(p); break;
        case 128: paged_score_kernel<E, 64, 2><<<blocks, 256, 0, st>>>(p); break;
        case 256:  // (head dims up to 1024: more chunks are of wider types)
            if constexpr (sizeof(E) > 1) paged_score_kernel<E, 64, 4><<<blocks, 256, 0, st>>>(p);
            break;
        default:
            if constexpr (sizeof(E) > 2) paged_score_kernel<E, 64, 8><<<blocks, 256, 0, st>>>(p);
            break;
    }
    return status_from_launch();
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
    p.splits = splits_for(static_cast<int64_t>(B) * Hkv, max_pages);
    const int64_t units = static_cast<int64_t>(B) * Hkv * p.splits;
    const unsigned blocks = static_cast<unsigned>((units + 3) / 4);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int lpr = std::min(64, pow2_up(D / n));
    if (cache_dtype == SA_BF16) return launch_bounds<bf16>(p, lpr, blocks, st);
    if (cache_dtype == SA_F16) return launch_bounds<f16>(p, lpr, blocks, st);
    if (cache_dtype == SA_F32) return launch_bounds<float>(p, lpr, blocks, st);
    return launch_bounds<fp8e4>(p, lpr, blocks, st);
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
    if (!q || !pages || !q_strides || !context_lens || (n_pages > 0 && max_pages > 0 && (!bounds || !block_table)))
        return SA_ERR_NULL_POINTER;
    const int q16 = dtype == SA_F32 ? 4 : 8;
    if (q_strides[3] != 1 || q_strides[0] % q16 != 0 || q_strides[1] % q16 != 0 || !aligned16(q) || !aligned16(bounds) || D % (16 / bytes_of(cache_dtype)) != 0) return SA_ERR_BAD_STRIDE;
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
    p.qcode = dtype;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (choose) {
        const int chunks = 2 * D * bytes_of(cache_dtype) / 16;
        const int lpp = std::min(64, pow2_up(chunks)), nch = pow2_up((chunks + lpp - 1) / lpp);
        const int batch = kBatch * (64 / lpp);  // pages that a wave takes at a time
        p.splits = splits_for(static_cast<int64_t>(B) * Hkv, (max_pages + batch - 1) / batch);
        const int64_t units = static_cast<int64_t>(B) * Hkv * p.splits;
        const unsigned blocks = static_cast<unsigned>((units + 3) / 4);
        const int status = cache_dtype == SA_BF16  ? launch_scores<bf16>(p, lpp, nch, blocks, st)
                           : cache_dtype == SA_F16 ? launch_scores<f16>(p, lpp, nch, blocks, st)
                           : cache_dtype == SA_F32 ? launch_scores<float>(p, lpp, nch, blocks, st)
                                                   : launch_scores<fp8e4>(p, lpp, nch, blocks, st);
        if (status != 0) return status;
    }
    const unsigned lists = static_cast<unsigned>(B) * Hkv;
    if (!choose || max_pages <= 512 * 2) paged_pick_kernel<512, 2><<<lists, 512, 0, st>>>(p);
    else if (max_pages <= 512 * 8) paged_pick_kernel<512, 8><<<lists, 512, 0, st>>>(p);
    else if (max_pages <= 1024 * 16) paged_pick_kernel<1024, 16><<<lists, 1024, 0, st>>>(p);
    else paged_pick_kernel<1024, 0><<<lists, 1024, 0, st>>>(p);
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
