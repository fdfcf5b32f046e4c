// pkv_paged.cuh -- what the kernels over a paged code cache share: the page descriptor on the
// device, how a sequence's tokens are found, and how attention work is cut into ranges.
#pragma once

#include <atomic>
#include <mutex>

#include "pkv_common.cuh"
#include "pkv_mma.cuh"

namespace pkv {

// The pages of a cache, strides in bytes.
struct Pages {
    const uint8_t *k, *v;
    int64_t page_bs, head_bs, tok_bs;
    const int32_t* table;
    int64_t table_stride;
    int num_pages, Hkv, ps_log2, B, max_pages;
};

__device__ __forceinline__ int clamp_len(const Pages& g, int len) {
    const int64_t cap = (int64_t)g.max_pages << g.ps_log2;
    return (int)min((int64_t)max(len, 0), cap);
}

// What a call reads -- its inputs and its codec's tables -- was written by earlier kernels of its stream, whose last one
// may still run when the call's first CTAs come up (launch_behind). A call's first kernel reads it by ordinary loads,
// which stay behind the grid dependency; the read-only path (__ldg) need not, and is for the tables in later kernels.
template <class T> __device__ __forceinline__ T input(const T* p) { return *p; }

// Physical page of logical page j of sequence b, or -1 (and the error word) when the table names none.
__device__ __forceinline__ int page_of(const Pages& g, int b, int j) {
    if ((unsigned)j >= (unsigned)g.max_pages) {
        flag_error(kErrPage);
        return -1;
    }
    const int page = input(g.table + (int64_t)b * g.table_stride + j);
    if ((unsigned)page >= (unsigned)g.num_pages) {
        flag_error(kErrPage);
        return -1;
    }
    return page;
}

__device__ __forceinline__ int64_t slot_offset(const Pages& g, int page, int hk, int r) {
    return (int64_t)page * g.page_bs + (int64_t)hk * g.head_bs + (int64_t)r * g.tok_bs;
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device: asked of the runtime once per device
// and growth (`seen`: the most asked for on each device, one array per kernel).
template <class K>
static int allow_smem(K kernel, int bytes, std::atomic<int> (&seen)[64]) {
    static std::mutex growing;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return PKV_ERR_CUDA;
    if (dev < 0 || dev >= 64) return PKV_ERR_UNSUPPORTED;
    if (seen[dev].load(std::memory_order_acquire) >= bytes) return PKV_OK;
    std::lock_guard<std::mutex> hold(growing);              // (a smaller request must not undo a larger one)
    if (seen[dev].load(std::memory_order_acquire) >= bytes) return PKV_OK;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return PKV_ERR_CUDA;
    seen[dev].store(bytes, std::memory_order_release);
    return PKV_OK;
}

// A launch whose CTAs may come up while the launch before it in the stream drains (programmatic dependent launch).
//  * The first kernel of a call waits for the grid dependency before it reads anything, and lets the next kernel come up
//    (triggers) only after that wait. So whatever ran before the call is complete when a later kernel of the call starts.
//  * A later kernel may therefore read the call's inputs and tables ahead of its own wait, but what the call's earlier
//    kernels write only behind it.
//  * No kernel writes outputs or workspace ahead of its wait, and every CTA waits before it ends.
template <class... A, class... B>
static int launch_behind(void (*kernel)(A...), unsigned ctas, int threads, size_t smem, int cluster, cudaStream_t st, B... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? PKV_OK : PKV_ERR_CUDA;
}

// ---- attention ---------------------------------------------------------------------------------
// A unit is NB blocks of four query heads of one (sequence, KV head); units are numbered sequence-major, block x of
// unit u is block u NB + x.  Its
// tokens are the sequence's (or the listed pages', in list order) in granules of what a warp takes at a time,
// 2^gran_log2 = 16 or 32.  The granules of all units form one line of T granules, cut among Gd CTAs: the grid, or
// where that is less one per unit or per 256 tokens, below which a CTA's warps would have little to share.  Two ways to cut:
//  * evenly: CTA c takes [c T / Gd, (c + 1) T / Gd), whatever the units.  Every CTA streams the same, but most
//    units end inside a CTA, which then sets up a second range (about 5 us).
//  * by units, while a CTA's share is below kUnitShare tokens (of which 512 take 2.7 us): a unit [a, e) goes
//    to the CTAs [s(a), s(e)), s(t) = round(t Gd / T), in equal parts, or whole to CTA s(a) when that is none.
// Each (CTA, unit) range leaves one partial softmax state; range (c, u) uses partial row c + u, so a
// unit's rows lie side by side.
constexpr int kUnitShare = 4096;

struct PagedParams {
    Pages pg;
    int G, NB, UG, UH, dim, m, cb, gran_log2;   // NB blocks of four heads to a unit, UG units per KV head, UH = Hkv UG
    const void* q; int qdt; int64_t q_bs, q_hs;
    const int32_t* seq_lens;
    const int32_t* selected; int n_sel;
    float scale_log2;
    void* out; int odt; int64_t out_bs, out_hs;
    const float* w_in; float* w_out; int64_t w_rs; int w_slots;
    const float *R, *dec_z, *dec_xy;
    int bits_z, bits_flat, xy_per_z;
    float* part;                               // [grid + units][NB][4][dim + 2]: m (log2 units), l, o
    uint32_t* frag; float* head;               // query operands, per-head numbers (paged_query_kernel)
    float* raw; int64_t raw_us; int raw_h;     // scores of every token, [block][token][raw_h]
    int grid, units;
};

__device__ __forceinline__ int granules_of(const PagedParams& p, int b) {
    const int n = p.selected ? p.n_sel << p.pg.ps_log2 : clamp_len(p.pg, input(p.seq_lens + b));
    return (n + (1 << p.gran_log2) - 1) >> p.gran_log2;
}

// Granules of the sequences before b, and of all of them (times UH: the line of all units).  Whole warps.
__device__ inline void granule_line(const PagedParams& p, int b, int64_t& before, int64_t& total) {
    int64_t sb = 0, st = 0;
    if (p.selected) {
        const int64_t n = (int64_t)granules_of(p, 0) * p.UH;
        before = n * b;
        total = n * p.pg.B;
        return;
    }
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < p.pg.B; i += 32) {
        const int n = granules_of(p, i);
        st += n;
        if (i < b) sb += n;
    }
    #pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        sb += __shfl_xor_sync(0xffffffffu, sb, off);
        st += __shfl_xor_sync(0xffffffffu, st, off);
    }
    before = sb * p.UH;
    total = st * p.UH;
}

struct PagedItem { int b, hk, unit, g0, g1, row; };     // granules [g0, g1) of the unit, partial row

struct PagedCut { int64_t total; int gd; bool by_unit; };

__device__ __forceinline__ PagedCut paged_cut(const PagedParams& p, int64_t total) {
    PagedCut c;
    c.total = total;
    const int64_t tokens = total << p.gran_log2;
    c.gd = (int)min((int64_t)p.grid, min(total, max((tokens + 255) / 256, (int64_t)p.units)));
    c.by_unit = tokens < (int64_t)kUnitShare * c.gd;
    return c;
}

// s(t) of the cut by units
__device__ __forceinline__ int unit_cut(const PagedCut& c, int64_t t) {
    return (int)((2 * t * c.gd + c.total) / (2 * c.total));
}

struct PagedCursor { PagedCut cut; int64_t t, end, base; int b; };

// Whole warps; every warp of the CTA walks the same items.
__device__ inline PagedCursor paged_begin(const PagedParams& p) {
    PagedCursor c;
    int64_t total, before;
    granule_line(p, 0, before, total);
    c.cut = paged_cut(p, total);
    c.b = 0;
    c.base = 0;
    const int64_t x = blockIdx.x, gd = c.cut.gd;
    if (x >= gd) {
        c.t = c.end = 0;
        return c;
    }
    if (c.cut.by_unit) {                                    // units that start or lie where s may be x
        c.t = max((int64_t)0, ((2 * x - 1) * total) / (2 * gd) - 1);
        c.end = total;
    } else {
        c.t = x * total / gd;
        c.end = (x + 1) * total / gd;
    }
    // the sequence of granule t: 32 sequences at a time
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < p.pg.B; b0 += 32) {
        const int64_t n = (b0 + lane < p.pg.B) ? (int64_t)granules_of(p, b0 + lane) * p.UH : 0;
        int64_t inc = n;
        #pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, inc, off);
            if (lane >= off) inc += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, c.base + inc > c.t);
        if (past) {
            const int f = __ffs(past) - 1;
            c.b = b0 + f;
            c.base += __shfl_sync(0xffffffffu, inc - n, f);
            break;
        }
        c.base += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (c.cut.by_unit) c.t -= (c.t - c.base) % granules_of(p, c.b);      // to the start of its unit
    return c;
}

__device__ inline bool paged_next(const PagedParams& p, PagedCursor& c, PagedItem& it) {
    const int x = blockIdx.x;
    while (c.t < c.end) {
        const int n = granules_of(p, c.b);
        const int64_t off = c.t - c.base;
        if (off >= (int64_t)n * p.UH) {
            c.base += (int64_t)n * p.UH;
            ++c.b;
            continue;
        }
        const int u = (int)(off / n);
        it.b = c.b;
        it.hk = u / p.UG;
        it.unit = c.b * p.UH + u;
        it.row = x + it.unit;
        if (c.cut.by_unit) {
            const int sa = min(unit_cut(c.cut, c.t), c.cut.gd - 1), k = max(1, unit_cut(c.cut, c.t + n) - sa);
            if (sa > x) {
                c.t = c.end;
                return false;
            }
            c.t += n;
            if (x >= sa + k) continue;
            it.g0 = (int)((int64_t)(x - sa) * n / k);
            it.g1 = (int)((int64_t)(x - sa + 1) * n / k);
        } else {
            it.g0 = (int)(off - (int64_t)u * n);
            it.g1 = (int)min((int64_t)n, it.g0 + (c.end - c.t));
            c.t += it.g1 - it.g0;
        }
        return true;
    }
    return false;
}

// The partial rows [r0, r1) of a unit, none without granules.  Whole warps.
__device__ inline void unit_rows(const PagedParams& p, int unit, int& r0, int& r1) {
    const int b = unit / p.UH, n = granules_of(p, b);
    int64_t before, total;
    granule_line(p, b, before, total);
    r0 = r1 = 0;
    if (n == 0) return;
    const PagedCut c = paged_cut(p, total);
    const int64_t a = before + (int64_t)(unit % p.UH) * n;
    if (c.by_unit) {
        const int sa = min(unit_cut(c, a), c.gd - 1);
        r0 = sa + unit;
        r1 = r0 + max(1, unit_cut(c, a + n) - sa);
    } else {
        r0 = (int)(((a + 1) * c.gd - 1) / total) + unit;
        r1 = (int)(((a + n) * c.gd - 1) / total) + unit + 1;
    }
}

// Page j of an attention range: the sequence's logical page (j itself, or entry j of its list) and the physical one;
// -1 for what is masked.
struct RangePage { int logical, page; };

__device__ __forceinline__ RangePage range_page(const PagedParams& p, int b, int hk, int j) {
    if (!p.selected) return {j, page_of(p.pg, b, j)};
    const int32_t* s = p.selected + ((int64_t)b * p.pg.Hkv + hk) * p.n_sel + j;
    const int lp = input(s), before = j > 0 ? input(s - 1) : -1;
    if (lp < 0) return {-1, -1};                            // padding
    if ((j > 0 && (before < 0 || before >= lp)) ||          // not ascending, or behind the sequence's end
        (int64_t)lp << p.pg.ps_log2 >= clamp_len(p.pg, input(p.seq_lens + b))) {
        flag_error(kErrPage);
        return {-1, -1};
    }
    return {lp, page_of(p.pg, b, lp)};
}

// bulk_g2s (pkv_common.cuh) to a shared address
__device__ __forceinline__ void bulk_g2s_at(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        :: "r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float load_any(const void* q, int dt, int64_t i) {
    if (dt == PKV_F32) return input(static_cast<const float*>(q) + i);
    if (dt == PKV_BF16) return __bfloat162float(input(static_cast<const __nv_bfloat16*>(q) + i));
    return __half2float(input(static_cast<const __half*>(q) + i));
}

__device__ __forceinline__ void store_any(void* o, int dt, int64_t i, float v) {
    if (dt == PKV_F32) Elem<PKV_F32>::store(static_cast<float*>(o) + i, v);
    else if (dt == PKV_BF16) Elem<PKV_BF16>::store(static_cast<__nv_bfloat16*>(o) + i, v);
    else Elem<PKV_F16>::store(static_cast<__half*>(o) + i, v);
}

}  // namespace pkv
