// Pages, block tables and slot maps of a serving step, from the sequences'
// lengths, on the device: a step needs no copy of its lengths to the host.
//
// The free pages are a stack: free_pages[0 .. n_free).  For sequence b with
// ctx_b tokens and new_b to come, in the order of the sequences:
//   start_b  = min(sum_{b' < b} new_b', n_tokens)       (packed position of its first new token)
//   want_b   = min(ctx_b + start_{b+1} - start_b, table width * P)
//   had_b    = ceil(ctx_b / P),  need_b = ceil(want_b / P) - had_b
//   before_b = sum_{b' < b} need_b',  got_b = min(need_b, max(0, n_free - before_b))
//   len_b    = min(want_b, (had_b + got_b) P)
// A sequence that cannot have all its pages is cut to those that are left, and
// its new length says so.  New page j of b is free_pages[n_free - 1 -
// (before_b + j)].  Token i of the packed tokens belongs to the b with
// start_b <= i < start_{b+1}, at position ctx_b + i - start_b; its slot is
// page * P + row, or -1 past len_b.
//
// One launch: every block works out the sums for itself (they are a few
// thousand numbers), and a new page's first token, whose thread knows the page
// anyway, enters it into the table.  The entries that are read (below had_b)
// are never the ones that are written.  Bound by the launch and a chain of loads
// and sums: 3.6 us for a token of each of 64 sequences, 5.7 for 67600 tokens of
// 256.
#include "common.hpp"

namespace sa {
namespace {

constexpr int kMaxSeqs = 4096;  // their sums lie in LDS
constexpr int kThreads = 256;

struct ReserveParams {
    int32_t* table;
    const int32_t* ctx;
    const int32_t* fresh;
    const int32_t* free_pages;
    const int32_t* n_free;
    int32_t *slots, *positions, *sequences, *starts, *lens, *n_free_out;
    int64_t bt_stride;
    int B, W, P, n_tokens, n_pages;
};

// Inclusive prefix sum over the block's threads; total: the sum of all.
__device__ __forceinline__ int64_t block_prefix(int64_t v, int64_t* part, int64_t& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t u = __shfl_up(v, off);
        if (lane >= off) v += u;
    }
    __syncthreads();  // (the last call's sums have been read)
    if (lane == 63) part[wv] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
        if (i < wv) before += part[i];
        total += part[i];
    }
    return v + before;
}

__global__ __launch_bounds__(kThreads) void paged_reserve_kernel(ReserveParams p) {
    __shared__ int32_t starts[kMaxSeqs + 1];
    __shared__ int32_t before[kMaxSeqs];
    __shared__ int64_t part[kThreads / 64];
    const int64_t cap = static_cast<int64_t>(p.W) * p.P;
    const int avail = min(max(p.n_free[0], 0), p.n_pages);
    int64_t tokens = 0, pages = 0;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int64_t ctx = 0, fresh = 0, total;
        if (b < p.B) {
            ctx = smaller<int64_t>(larger<int64_t>(p.ctx[b], 0), cap);
            fresh = max(p.fresh[b], 0);
        }
        const int64_t end = tokens + block_prefix(fresh, part, total);
        tokens += total;
        const int64_t s0 = smaller<int64_t>(end - fresh, p.n_tokens);
        const int64_t s1 = smaller<int64_t>(end, p.n_tokens);
        const int64_t want = smaller<int64_t>(ctx + s1 - s0, cap);
        const int64_t had = (ctx + p.P - 1) / p.P;
        const int64_t need = b < p.B ? (want + p.P - 1) / p.P - had : 0;
        const int64_t bef = pages + block_prefix(need, part, total) - need;
        pages += total;
        if (b < p.B) {
            starts[b] = static_cast<int32_t>(s0);
            before[b] = static_cast<int32_t>(smaller<int64_t>(bef, INT32_MAX));
            if (blockIdx.x == 0) {
                const int64_t got = smaller<int64_t>(larger<int64_t>(avail - bef, 0), need);
                p.starts[b] = static_cast<int32_t>(s0);
                p.lens[b] = static_cast<int32_t>(smaller<int64_t>(want, (had + got) * p.P));
            }
        }
    }
    const int32_t last = static_cast<int32_t>(smaller<int64_t>(tokens, p.n_tokens));
    if (threadIdx.x == 0) {
        starts[p.B] = last;
        if (blockIdx.x == 0) {
            p.starts[p.B] = last;
            p.n_free_out[0] = static_cast<int32_t>(avail - smaller<int64_t>(pages, avail));
        }
    }
    __syncthreads();
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= p.n_tokens) return;
    int slot = -1, pos = 0, seq = -1;
    if (i < last) {
        int lo = 0, hi = p.B;  // starts[lo] <= i < starts[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= i) lo = mid;
            else hi = mid;
        }
        seq = lo;
        const int ctx = static_cast<int>(smaller<int64_t>(larger<int64_t>(p.ctx[seq], 0), cap));
        const int64_t at = static_cast<int64_t>(ctx) + i - starts[seq];
        pos = static_cast<int>(smaller<int64_t>(at, INT32_MAX));
        if (at < cap) {
            const int had = (ctx + p.P - 1) / p.P;
            const int pi = pos / p.P, row = pos - pi * p.P;
            int page = -1;
            if (pi < had) {
                page = p.table[seq * p.bt_stride + pi];
            } else {
                const int64_t taken = static_cast<int64_t>(before[seq]) + pi - had;
                if (taken < avail) {
                    page = p.free_pages[avail - 1 - taken];
                    if (row == 0) p.table[seq * p.bt_stride + pi] = page;
                }
            }
            if (page >= 0 && page < p.n_pages) slot = page * p.P + row;
        }
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
    p.sequences[i] = seq;
}

// Pages of the finished sequences, pushed on the free stack in the order of the
// sequences and their tables.  Table entries that name no page are skipped, and
// those given back are set to -1, so giving a sequence back twice gives nothing
// the second time.  Two launches: the pages of each sequence are counted, then
// every block adds up those before its own.
struct ReleaseParams {
    int32_t* table;
    const int32_t* ctx;
    const uint8_t* finished;
    int32_t* free_pages;
    const int32_t* n_free;
    int32_t *lens, *n_free_out, *counts;
    int64_t bt_stride;
    int B, W, P, n_pages;
};

__device__ __forceinline__ int pages_of(const ReleaseParams& p, int b) {
    if (!p.finished[b]) return 0;
    const int64_t cap = static_cast<int64_t>(p.W) * p.P;
    return static_cast<int>((smaller<int64_t>(larger<int64_t>(p.ctx[b], 0), cap) + p.P - 1) / p.P);
}

// A block takes a sequence, kRun entries a thread at once: waiting for a table
// of 1024 entries 64 at a time made 7 us of either kernel.
constexpr int kRun = 4;

__device__ __forceinline__ void read_entries(const ReleaseParams& p, int b, int j0, int n, int* page) {
    const int32_t* row = p.table + b * p.bt_stride;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int j = j0 + i * kThreads + static_cast<int>(threadIdx.x);
        page[i] = j < n ? row[j] : -1;
    }
}

__global__ __launch_bounds__(kThreads) void paged_release_count_kernel(ReleaseParams p) {
    __shared__ int part[kThreads / 64];
    const int b = blockIdx.x;
    const int n = pages_of(p, b);
    int found = 0;  // of the wave
    for (int j0 = 0; j0 < n; j0 += kRun * kThreads) {
        int page[kRun];
        read_entries(p, b, j0, n, page);
#pragma unroll
        for (int i = 0; i < kRun; ++i) found += __popcll(__ballot(page[i] >= 0 && page[i] < p.n_pages));
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = found;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 64; ++i) all += part[i];
        p.counts[b] = all;
    }
}

__global__ __launch_bounds__(kThreads) void paged_release_kernel(ReleaseParams p) {
    __shared__ int words[kRun * kThreads / 64];  // pages given back in each 64 entries
    const int b = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int n = pages_of(p, b);
    if (n == 0 && b != 0) {  // (the first block also says how many pages there are)
        if (threadIdx.x == 0) p.lens[b] = p.finished[b] ? 0 : p.ctx[b];
        return;
    }
    int64_t before = 0, all = 0;  // pages of the sequences before this one, and of all
    for (int i = lane; i < p.B; i += 64) {
        const int c = p.counts[i];
        all += c;
        if (i < b) before += c;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        before += __shfl_xor(before, o);
        all += __shfl_xor(all, o);
    }
    const int base = min(max(p.n_free[0], 0), p.n_pages);
    if (threadIdx.x == 0) {
        p.lens[b] = p.finished[b] ? 0 : p.ctx[b];
        if (b == 0) p.n_free_out[0] = static_cast<int32_t>(smaller<int64_t>(base + all, p.n_pages));
    }
    int64_t at = base + before;
    for (int j0 = 0; j0 < n; j0 += kRun * kThreads) {
        int page[kRun];
        read_entries(p, b, j0, n, page);
        unsigned long long back[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            back[i] = __ballot(page[i] >= 0 && page[i] < p.n_pages);
            if (lane == 0) words[i * (kThreads / 64) + wv] = __popcll(back[i]);
        }
        __syncthreads();
        int64_t to[kRun], sum = 0;
#pragma unroll
        for (int w = 0; w < kRun * kThreads / 64; ++w) {  // (the words are in the entries' order)
            if (w % (kThreads / 64) == wv) to[w / (kThreads / 64)] = at + sum;
            sum += words[w];
        }
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int j = j0 + i * kThreads + static_cast<int>(threadIdx.x);
            const int64_t slot = to[i] + __popcll(back[i] & ((1ull << lane) - 1));
            if ((back[i] >> lane & 1) && slot < p.n_pages) p.free_pages[slot] = page[i];
            if (j < n) p.table[b * p.bt_stride + j] = -1;
        }
        at += sum;
        __syncthreads();  // (words have been read)
    }
}

int check_maps(int B, int W, int P, int n_pages, int64_t bt_stride) {
    if (B < 0 || W < 0 || P <= 0 || n_pages < 0) return SA_ERR_BAD_SHAPE;
    if (B > kMaxSeqs) return SA_ERR_UNSUPPORTED;
    // slots and lengths are 32-bit
    if (static_cast<int64_t>(n_pages) * P > INT32_MAX || static_cast<int64_t>(W) * P > INT32_MAX) return SA_ERR_BAD_SHAPE;
    return bt_stride < W ? SA_ERR_BAD_STRIDE : 0;
}

}  // namespace
}  // namespace sa

extern "C" int sa_paged_reserve(int32_t* block_table, const int32_t* context_lens, const int32_t* new_lens,
                                const int32_t* free_pages, const int32_t* n_free, int32_t* slots, int32_t* positions,
                                int32_t* sequences, int32_t* starts, int32_t* lens_out, int32_t* n_free_out, int B,
                                int max_pages, int page_size, int n_pages, int n_tokens, int64_t bt_stride,
                                sa_stream_t stream) {
    using namespace sa;
    const int chk = check_maps(B, max_pages, page_size, n_pages, bt_stride);
    if (chk != 0) return chk;
    if (n_tokens < 0) return SA_ERR_BAD_SHAPE;
    if (!n_free || !starts || !n_free_out || (B > 0 && (!context_lens || !new_lens || !lens_out)) ||
        (B > 0 && max_pages > 0 && !block_table) || (n_pages > 0 && !free_pages) ||
        (n_tokens > 0 && (!slots || !positions || !sequences)))
        return SA_ERR_NULL_POINTER;
    ReserveParams p{};
    p.table = block_table;
    p.ctx = context_lens;
    p.fresh = new_lens;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.slots = slots;
    p.positions = positions;
    p.sequences = sequences;
    p.starts = starts;
    p.lens = lens_out;
    p.n_free_out = n_free_out;
    p.bt_stride = bt_stride;
    p.B = B;
    p.W = max_pages;
    p.P = page_size;
    p.n_tokens = n_tokens;
    p.n_pages = n_pages;
    const int64_t blocks = n_tokens == 0 ? 1 : (static_cast<int64_t>(n_tokens) + kThreads - 1) / kThreads;
    paged_reserve_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(p);
    return status_from_launch();
}

extern "C" int sa_paged_release(int32_t* block_table, const int32_t* context_lens, const uint8_t* finished,
                                int32_t* free_pages, const int32_t* n_free, int32_t* lens_out, int32_t* n_free_out,
                                int32_t* counts_ws, int B, int max_pages, int page_size, int n_pages,
                                int64_t bt_stride, sa_stream_t stream) {
    using namespace sa;
    const int chk = check_maps(B, max_pages, page_size, n_pages, bt_stride);
    if (chk != 0) return chk;
    if (B == 0) return SA_ERR_BAD_SHAPE;  // (nothing would write n_free_out)
    if (!context_lens || !finished || !n_free || !lens_out || !n_free_out || !counts_ws ||
        (max_pages > 0 && !block_table) || (n_pages > 0 && !free_pages))
        return SA_ERR_NULL_POINTER;
    ReleaseParams p{};
    p.table = block_table;
    p.ctx = context_lens;
    p.finished = finished;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.lens = lens_out;
    p.n_free_out = n_free_out;
    p.counts = counts_ws;
    p.bt_stride = bt_stride;
    p.B = B;
    p.W = max_pages;
    p.P = page_size;
    p.n_pages = n_pages;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    paged_release_count_kernel<<<static_cast<unsigned>(B), kThreads, 0, st>>>(p);
    const int status = status_from_launch();
    if (status != 0) return status;
    paged_release_kernel<<<static_cast<unsigned>(B), kThreads, 0, st>>>(p);
    return status_from_launch();
}
