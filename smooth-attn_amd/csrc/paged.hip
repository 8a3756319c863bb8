// Paged single-token squareplus decode through a block table (gfx950).
//
// out[b, h] = sum_{t < ctx_b} y_t V_t / (sum_t y_t + 1e-12),
// y_t = squareplus(2 scale q . K_t - 1)^2,
// K_t = k_cache[block_table[b, t / P], h / G, t % P]
//   (reference kernels.py:2681-2773 and the decode references of
//    tests/test_paged_long_context.py:39-65)
//
// Work split (stream-K style, balanced whatever the context lengths): a plan
// counts each sequence's 32-token tiles, prefix-sums them over (sequence, KV
// head) in that order and fixes the number of active waves Ne (every wave
// works it out, or for large batches a kernel: WavePlan); a persistent grid of one-wave blocks then gives wave w the tiles
// [floor(w Tt / Ne), floor((w+1) Tt / Ne)) of the Tt in total.  A wave's
// range is cut at (sequence, KV head) boundaries into pieces; each piece is
// walked in tiles of 32 tokens, reading every K/V row once for all G query
// heads that share the KV head (the reference grid (B, Hq) rereads each
// page G times).  Tiles are fetched with coalesced 16-byte loads (one 1 KB
// span per instruction) one tile ahead of the compute and staged in
// wave-private LDS.  Scores are S^T = K Q^T on MFMA with the G query heads
// as columns; the squareplus weights land in the B-operand layout of
// O^T += V^T P^T, and V^T comes from the row-major LDS tile through the
// transposing LDS read (see flash_common.hpp).  Each piece writes its
// unnormalised partial (O, S) into slot k of its (sequence, query head),
// k = its wave minus the wave that owns the segment's first tile; a merge
// kernel sums the slots in order (squareplus needs no running maximum, so
// merging is a plain sum) and divides once.
#include <atomic>
#include <mutex>

#include "paged_kernel.hpp"

namespace sa {
namespace {

// Workspace layout: plan (B + 2 int32, padded to 16 bytes), then the O and S
// partials (fp32).
int64_t plan_bytes(int B) { return ((static_cast<int64_t>(B) + 2) * 4 + 15) / 16 * 16; }

int64_t workspace_bytes_for(int B, int Hq, int D, int max_pages, int page_size, int per) {
    const int64_t slots = static_cast<int64_t>(B) * Hq * slots_for(max_pages, page_size, per);
    return plan_bytes(B) + slots * (D + 1) * static_cast<int64_t>(sizeof(float));
}

// The minimum tiles per active wave a launch uses: the workspace is sized
// for split_floor, and the launch takes the larger split its B * Hkv
// segments give (so its slots always fit).
int launch_per(int B, int Hq, int Hkv, int max_pages, int page_size) {
    return std::max(split_floor(B, Hq, max_pages, page_size),
                    split_for(static_cast<int64_t>(B) * Hkv, max_pages, page_size));
}

// Plan, partial and merge launches with the workspace at `ws` (laid out for
// `per` minimum tiles per wave).
int run_paged(const void* q, const void* k_cache, const void* v_cache, void* out, const int32_t* block_table,
              const int32_t* context_lens, int B, int Hq, int Hkv, int D, int page_size, int max_pages,
              int n_pages, const int64_t* q_strides, const int64_t* kv_strides, const int64_t* vv_strides,
              const int64_t* o_strides, int64_t bt_stride, float scale, int dtype, float* ws, int per,
              hipStream_t st) {
    PagedParams prm{};
    prm.q = q;
    prm.k = k_cache;
    prm.v = v_cache;
    prm.out = static_cast<bf16*>(out);
    prm.table = block_table;
    prm.ctx = context_lens;
    prm.per = per;
    prm.n_slots = static_cast<int>(slots_for(max_pages, page_size, per));
    prm.plan = reinterpret_cast<int*>(ws);
    prm.ws_o = ws + plan_bytes(B) / 4;
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
    prm.logP = __builtin_ctz(static_cast<unsigned>(page_size));
    prm.max_pages = max_pages;
    prm.n_pages = n_pages;
    prm.scale = scale;
    return launch_paged_types<false>(prm, dtype, st);
}

}  // namespace
}  // namespace sa

extern "C" int64_t sa_paged_decode_workspace_size(int B, int Hq, int D, int max_pages, int page_size) {
    if (B <= 0 || Hq <= 0 || D <= 0 || max_pages < 0 || page_size <= 0) return 0;
    return sa::workspace_bytes_for(B, Hq, D, max_pages, page_size, sa::split_floor(B, Hq, max_pages, page_size));
}

extern "C" int sa_paged_decode(const void* q, const void* k_cache, const void* v_cache, void* out,
                               const int32_t* block_table, const int32_t* context_lens, int B, int Hq, int Hkv,
                               int D, int page_size, int max_pages, int n_pages, const int64_t* q_strides,
                               const int64_t* kv_strides, const int64_t* vv_strides, const int64_t* o_strides,
                               int64_t bt_stride, float scale, int dtype, float* workspace, int64_t workspace_bytes,
                               sa_stream_t stream) {
    using namespace sa;
    const int chk = validate_paged(q, k_cache, v_cache, out, block_table, context_lens, B, Hq, Hkv, D, page_size,
                                   max_pages, n_pages, q_strides, kv_strides, vv_strides, o_strides, dtype);
    if (chk != 0) return chk > 0 ? 0 : chk;
    if (!workspace) return SA_ERR_NULL_POINTER;
    if (workspace_bytes < sa_paged_decode_workspace_size(B, Hq, D, max_pages, page_size)) return SA_ERR_WORKSPACE;
    return run_paged(q, k_cache, v_cache, out, block_table, context_lens, B, Hq, Hkv, D, page_size, max_pages,
                     n_pages, q_strides, kv_strides, vv_strides, o_strides, bt_stride, scale, dtype, workspace,
                     launch_per(B, Hq, Hkv, max_pages, page_size), reinterpret_cast<hipStream_t>(stream));
}

// ---------------------------------------------------------------------------
// Allocation-free decode.  The plan and partials live in `scratch`, a
// module-scope device array: each device that loads this library holds its
// own copy (SA_PAGED_NOALLOC_SCRATCH_BYTES) until the process ends.  In host
// code the array's name is only a host-side stand-in, so its device address
// is looked up once per device with hipGetSymbolAddress (with that device
// current) and that address is what the kernels receive.
// ---------------------------------------------------------------------------
static __device__ __align__(256) float scratch[SA_PAGED_NOALLOC_SCRATCH_BYTES / sizeof(float)];

namespace sa {
namespace {

constexpr int kMaxDevices = 64;
std::atomic<float*> g_scratch[kMaxDevices];
std::mutex g_scratch_mu;

// The current device's copy of `scratch` (0 = ok, else a status).
int scratch_of_current_device(float** out) {
    int dev = -1;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return static_cast<int>(e);
    if (dev < 0 || dev >= kMaxDevices) return SA_ERR_UNSUPPORTED;
    float* p = g_scratch[dev].load(std::memory_order_acquire);
    if (p == nullptr) {
        std::lock_guard<std::mutex> lock(g_scratch_mu);
        p = g_scratch[dev].load(std::memory_order_relaxed);
        if (p == nullptr) {
            void* addr = nullptr;
            const hipError_t es = hipGetSymbolAddress(&addr, HIP_SYMBOL(scratch));
            if (es != hipSuccess) return static_cast<int>(es);
            if (addr == nullptr) return SA_ERR_WORKSPACE;
            p = static_cast<float*>(addr);
            g_scratch[dev].store(p, std::memory_order_release);
        }
    }
    *out = p;
    return 0;
}

}  // namespace
}  // namespace sa

extern "C" int sa_paged_decode_noalloc(const void* q, const void* k_cache, const void* v_cache, void* out,
                                       const int32_t* block_table, const int32_t* context_lens, int B, int Hq,
                                       int Hkv, int D, int page_size, int max_pages, int n_pages,
                                       const int64_t* q_strides, const int64_t* kv_strides,
                                       const int64_t* vv_strides, const int64_t* o_strides, int64_t bt_stride,
                                       float scale, int dtype, sa_stream_t stream) {
    using namespace sa;
    const int chk = validate_paged(q, k_cache, v_cache, out, block_table, context_lens, B, Hq, Hkv, D, page_size,
                                   max_pages, n_pages, q_strides, kv_strides, vv_strides, o_strides, dtype);
    if (chk != 0) return chk > 0 ? 0 : chk;
    // The workspace launch's split, or a coarser one (more tiles per wave,
    // fewer partial slots) when its partials would not fit the scratch: the
    // plan honours any per, which only caps how many waves share the work.
    int per = launch_per(B, Hq, Hkv, max_pages, page_size);
    constexpr int64_t cap = SA_PAGED_NOALLOC_SCRATCH_BYTES;
    while (workspace_bytes_for(B, Hq, D, max_pages, page_size, per) > cap &&
           slots_for(max_pages, page_size, per) > 2)
        per *= 2;
    if (workspace_bytes_for(B, Hq, D, max_pages, page_size, per) > cap) return SA_ERR_WORKSPACE;
    float* ws = nullptr;
    const int sst = scratch_of_current_device(&ws);
    if (sst != 0) return sst;
    return run_paged(q, k_cache, v_cache, out, block_table, context_lens, B, Hq, Hkv, D, page_size, max_pages,
                     n_pages, q_strides, kv_strides, vv_strides, o_strides, bt_stride, scale, dtype, ws, per,
                     reinterpret_cast<hipStream_t>(stream));
}
