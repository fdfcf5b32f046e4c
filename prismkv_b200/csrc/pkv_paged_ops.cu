// pkv_paged_ops.cu -- the kernels around attention over a paged code cache: storing rows, page
// summaries, choosing pages, choosing tokens to keep, and moving them.

#include <climits>

#include <cooperative_groups.h>

#include "pkv_paged.cuh"

namespace pkv {
namespace cg = cooperative_groups;

// ---- copies of code rows ------------------------------------------------------------------------
// One row of m codes = `bytes` bytes: 16-byte pieces, the last one short when bytes % 16 != 0 (rows
// start on 16-byte boundaries).  Piece i of a row, src and dst at the rows' starts:
__device__ __forceinline__ void copy_piece(uint8_t* dst, const uint8_t* src, int bytes, int i) {
    const int at = i * 16;
    if (at + 16 <= bytes) {
        *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
    } else {
        for (int x = at; x < bytes; ++x) dst[x] = src[x];
    }
}

// Rows (b, hk, i) of contiguous codes (any alignment of two bytes) into slots start[b] + i.
__global__ void pages_store_kernel(Pages g, uint8_t* dst, const uint8_t* codes, int bytes, int n,
                                   const int32_t* start, const int32_t* counts) {
    const int64_t rows = (int64_t)g.B * g.Hkv * n;
    const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;   // eight threads a row
    if (row >= rows) return;
    const int i = (int)(row % n), hk = (int)(row / n % g.Hkv), b = (int)(row / n / g.Hkv);
    if (counts && i >= counts[b]) return;
    const int64_t t = (int64_t)start[b] + i;
    if (t < 0 || t >= ((int64_t)g.max_pages << g.ps_log2)) {
        flag_error(kErrPage);
        return;
    }
    const int page = page_of(g, b, (int)(t >> g.ps_log2));
    if (page < 0) return;
    uint8_t* d = dst + slot_offset(g, page, hk, (int)(t & ((1 << g.ps_log2) - 1)));
    const uint8_t* s = codes + row * bytes;
    for (int x = threadIdx.x & 7; x < bytes; x += 8) d[x] = s[x];
}

// Slots kept[b, hk, i] of the source pages into slots i of the destination's, K and V.  One thread per
// 16-byte piece of a row; nothing is read twice, so the copies' bytes bound it.
__global__ void tokens_gather_kernel(Pages s, Pages d, uint8_t* dk, uint8_t* dv, int bytes, const int32_t* kept,
                                     int keep) {
    const int pieces = (bytes + 15) / 16;
    const int64_t total = (int64_t)s.B * s.Hkv * keep * pieces;
    for (int64_t x = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; x < total; x += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = x / pieces;
        const int pc = (int)(x - row * pieces);
        const int i = (int)(row % keep), bh = (int)(row / keep), hk = bh % s.Hkv, b = bh / s.Hkv;
        const int t = __ldg(kept + row);
        if (t < 0) continue;
        const int sp = page_of(s, b, t >> s.ps_log2), dp = page_of(d, b, i >> d.ps_log2);
        if (sp < 0 || dp < 0) continue;
        const int64_t so = slot_offset(s, sp, hk, t & ((1 << s.ps_log2) - 1));
        const int64_t to = slot_offset(d, dp, hk, i & ((1 << d.ps_log2) - 1));
        copy_piece(dk + to, s.k + so, bytes, pc);
        copy_piece(dv + to, s.v + so, bytes, pc);
    }
}

// ---- page summaries -------------------------------------------------------------------------------
// Per page, KV head and channel the least and greatest grid value of the page's tokens; a step is 128
// grid values, so the floor is a shift and the ceiling a shift of the value + 127.  One warp per (page,
// KV head), lanes over triplets.
struct SummaryParams {
    Pages pg;
    const int32_t *seq_lens, *start;
    const int16_t *grid_z, *grid_xy;
    int8_t* out;
    int m, cb, pitch, bits_flat, code_mask;
};

__global__ void __launch_bounds__(256) pages_summarize_kernel(SummaryParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (w >= (int64_t)p.pg.B * p.pg.max_pages * p.pg.Hkv) return;
    const int hk = (int)(w % p.pg.Hkv), j = (int)(w / p.pg.Hkv % p.pg.max_pages), b = (int)(w / p.pg.Hkv / p.pg.max_pages);
    const int L = clamp_len(p.pg, p.seq_lens[b]);
    const int t0 = j << p.pg.ps_log2, n = min(L - t0, 1 << p.pg.ps_log2);
    if (n <= 0 || (p.start && t0 + n <= p.start[b])) return;
    const int page = page_of(p.pg, b, j);
    if (page < 0) return;
    int8_t* o = p.out + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch;
    for (int i = lane; i < p.m; i += 32) {
        int lo[3] = {1 << 20, 1 << 20, 1 << 20}, hi[3] = {-(1 << 20), -(1 << 20), -(1 << 20)};
        for (int r = 0; r < n; ++r) {
            const uint8_t* row = p.pg.k + slot_offset(p.pg, page, hk, r);
            const int c = (p.cb == 1 ? row[i] : reinterpret_cast<const uint16_t*>(row)[i]) & p.code_mask;
            const int v[3] = {p.grid_z[c >> p.bits_flat], p.grid_xy[2 * c], p.grid_xy[2 * c + 1]};
            #pragma unroll
            for (int x = 0; x < 3; ++x) {
                lo[x] = min(lo[x], v[x]);
                hi[x] = max(hi[x], v[x]);
            }
        }
        #pragma unroll
        for (int x = 0; x < 3; ++x) {
            o[3 * i + x] = (int8_t)(lo[x] >> 7);
            o[p.pitch + 3 * i + x] = (int8_t)((hi[x] + 127) >> 7);
        }
    }
    for (int d = 3 * p.m + lane; d < p.pitch; d += 32) o[d] = o[p.pitch + d] = 0;
}

// ---- the k largest of a row, in index order ---------------------------------------------------------
// A cluster of CTAs holds a row of n keys (unsigned, larger = better), CTA `rank` the slice [lo, hi).
// Three digit passes (11, 11, 10 bits) of histograms narrow the k-th largest key; a last pass writes the
// indexes of the keys above it and of the first equal ones, in index order.  Counters of all CTAs meet in
// rank 0's shared memory.
constexpr int kTopThreads = 512;
constexpr int kTopBins = 2048;

struct TopShared {
    uint32_t hist[kTopBins];
    uint32_t warp[2][kTopThreads / 32];
    uint32_t bin, need;
};

template <class Key, class Put>
__device__ void top_row(TopShared& s, int lo, int hi, int n, int k, Key key, Put put) {
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rank = cl.block_rank(), C = cl.num_blocks();
    TopShared* s0 = cl.map_shared_rank(&s, 0);
    cl.sync();                                              // every CTA of the cluster runs: its memory may be reached
    uint32_t prefix = 0, need = (uint32_t)min(k, n);        // keys still to take among those with this prefix
    const bool all = n <= k;
    int shift = 32;
    if (!all) {
        #pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10, bins = 1 << bits;
            const uint32_t above = shift == 32 ? 0u : prefix >> shift;
            for (int i = tid; i < kTopBins; i += kTopThreads) s.hist[i] = 0;
            cl.sync();
            for (int i = lo + tid; i < hi; i += kTopThreads) {
                const uint32_t x = key(i);
                if (shift == 32 || (x >> shift) == above) atomicAdd(&s.hist[(x >> (shift - bits)) & (bins - 1)], 1u);
            }
            cl.sync();
            if (rank != 0)
                for (int i = tid; i < bins; i += kTopThreads)
                    if (s.hist[i]) atomicAdd(&s0->hist[i], s.hist[i]);
            cl.sync();
            // rank 0: the bin where the count from the top reaches `need`
            if (rank == 0) {
                const int per = bins / kTopThreads;         // 4 or 2 bins a thread, thread 0 the top ones
                uint32_t v[4], sum = 0;
                for (int j = 0; j < per; ++j) sum += v[j] = s.hist[bins - 1 - (tid * per + j)];
                uint32_t inc = sum;
                #pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t o = __shfl_up_sync(0xffffffffu, inc, off);
                    if (lane >= off) inc += o;
                }
                if (lane == 31) s.warp[0][warp] = inc;
                __syncthreads();
                for (int w = 0; w < warp; ++w) inc += s.warp[0][w];
                uint32_t cum = inc - sum;
                for (int j = 0; j < per; ++j) {
                    if (cum < need && cum + v[j] >= need) {
                        s.bin = bins - 1 - (tid * per + j);
                        s.need = need - cum;
                    }
                    cum += v[j];
                }
            }
            cl.sync();
            shift -= bits;
            prefix |= s0->bin << shift;
            need = s0->need;
            cl.sync();
        }
    }
    // counts of this slice
    uint32_t above = 0, equal = 0;
    for (int i = lo + tid; i < hi; i += kTopThreads) {
        const uint32_t x = key(i);
        above += all || x > prefix;
        equal += !all && x == prefix;
    }
    #pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        above += __shfl_xor_sync(0xffffffffu, above, off);
        equal += __shfl_xor_sync(0xffffffffu, equal, off);
    }
    __syncthreads();
    if (lane == 0) { s.warp[0][warp] = above; s.warp[1][warp] = equal; }
    __syncthreads();
    if (tid == 0) {
        uint32_t a = 0, e = 0;
        for (int w = 0; w < kTopThreads / 32; ++w) { a += s.warp[0][w]; e += s.warp[1][w]; }
        s0->hist[2 * rank] = a;                              // the histogram is done with
        s0->hist[2 * rank + 1] = e;
    }
    cl.sync();
    uint32_t base_a = 0, base_e = 0;
    for (unsigned r = 0; r < rank; ++r) { base_a += s0->hist[2 * r]; base_e += s0->hist[2 * r + 1]; }
    cl.sync();                                               // remote reads done before anyone leaves
    // in index order, kTopThreads keys at a time: position = keys above before + equal ones taken before
    for (int i0 = lo; i0 < hi; i0 += kTopThreads) {
        const int i = i0 + tid;
        const uint32_t x = i < hi ? key(i) : 0u;
        const bool a = i < hi && (all || x > prefix), e = i < hi && !all && x == prefix;
        const unsigned ma = __ballot_sync(0xffffffffu, a), me = __ballot_sync(0xffffffffu, e);
        __syncthreads();
        if (lane == 0) { s.warp[0][warp] = __popc(ma); s.warp[1][warp] = __popc(me); }
        __syncthreads();
        uint32_t pa = base_a, pe = base_e, ta = 0, te = 0;
        for (int w = 0; w < kTopThreads / 32; ++w) {
            if (w < warp) { pa += s.warp[0][w]; pe += s.warp[1][w]; }
            ta += s.warp[0][w];
            te += s.warp[1][w];
        }
        const unsigned below = (1u << lane) - 1u;
        pa += __popc(ma & below);
        pe += __popc(me & below);
        if (a || (e && pe < need)) put((int)(pa + min(pe, need)), i);
        base_a += ta;
        base_e += te;
    }
}

// this CTA's slice of n keys
__device__ __forceinline__ void top_slice(int n, int& lo, int& hi) {
    cg::cluster_group cl = cg::this_cluster();
    const int per = (n + (int)cl.num_blocks() - 1) / (int)cl.num_blocks();
    lo = min(n, (int)cl.block_rank() * per);
    hi = min(n, lo + per);
}

// ---- choosing pages ---------------------------------------------------------------------------------
struct SelectParams {
    Pages pg;
    const void* q; int qdt; int64_t q_bs, q_hs;
    int G, dim, pitch;
    const float* R;
    const int32_t* seq_lens;
    const int8_t* sums;
    int top, sinks, recent;
    int32_t* out;
};

__global__ void __launch_bounds__(kTopThreads) pages_select_kernel(SelectParams p) {
    extern __shared__ __align__(16) uint8_t ssm[];
    __shared__ TopShared top;
    __shared__ double amax_w[kTopThreads / 32];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, dim = p.dim;
    const int bh = blockIdx.x / cl.num_blocks(), b = bh / p.pg.Hkv, hk = bh % p.pg.Hkv;
    const int words = p.pitch / 4;
    double* sq = reinterpret_cast<double*>(ssm);                       // [G][dim]
    int8_t* qp = reinterpret_cast<int8_t*>(sq + p.G * dim);            // [G][pitch] positive, then negative parts
    uint32_t* keys = reinterpret_cast<uint32_t*>(qp + 2 * p.G * p.pitch);
    const int L = clamp_len(p.pg, p.seq_lens[b]);
    const int n = (int)(((int64_t)L + (1 << p.pg.ps_log2) - 1) >> p.pg.ps_log2);
    int lo, hi;
    top_slice(n, lo, hi);
    // rotated queries in 64 bits: a rounding to int8 must not turn on how a sum was ordered
    double amax = 0.0;
    for (int i = tid; i < p.G * dim; i += kTopThreads) {
        const int h = i / dim, k = i % dim;
        const int64_t qo = b * p.q_bs + (int64_t)(hk * p.G + h) * p.q_hs;
        double a = 0.0;
        for (int d = 0; d < dim; ++d) a = fma((double)load_any(p.q, p.qdt, qo + d), (double)__ldg(p.R + k * dim + d), a);
        sq[i] = a;
        amax = fmax(amax, fabs(a));
        if (!(fabs(a) <= 1e300)) amax = INFINITY;
    }
    #pragma unroll
    for (int off = 16; off >= 1; off >>= 1) amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if ((tid & 31) == 0) amax_w[tid >> 5] = amax;
    __syncthreads();
    amax = 0.0;
    for (int w = 0; w < kTopThreads / 32; ++w) amax = fmax(amax, amax_w[w]);
    for (int i = tid; i < p.G * p.pitch; i += kTopThreads) {
        const int h = i / p.pitch, d = i % p.pitch;
        int v = 0;
        // a zero or non-finite group scores every page alike
        if (d < dim && amax > 0.0 && amax <= 1e300) v = (int)rint(sq[h * dim + d] * 127.0 / amax);
        qp[i] = (int8_t)max(v, 0);
        qp[p.G * p.pitch + i] = (int8_t)min(v, 0);
    }
    __syncthreads();
    const int* qpos = reinterpret_cast<const int*>(qp);
    const int* qneg = qpos + p.G * words;
    for (int j = lo + tid; j < hi; j += kTopThreads) {
        uint32_t key = 0xffffffffu;
        if (j >= p.sinks && j < n - p.recent) {
            const int page = page_of(p.pg, b, j);
            key = 0;
            if (page >= 0) {
                const int* least = reinterpret_cast<const int*>(p.sums + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch);
                int best = INT_MIN;
                for (int h = 0; h < p.G; ++h) {
                    int a = 0;
                    for (int w = 0; w < words; ++w) {
                        a = __dp4a(least[words + w], qpos[h * words + w], a);
                        a = __dp4a(least[w], qneg[h * words + w], a);
                    }
                    best = max(best, a);
                }
                key = (uint32_t)best ^ 0x80000000u;
            }
        }
        keys[j - lo] = key;
    }
    __syncthreads();
    int32_t* out = p.out + (int64_t)bh * p.top;
    for (int i = min(n, p.top) + cl.block_rank() * kTopThreads + tid; i < p.top; i += cl.num_blocks() * kTopThreads) out[i] = -1;
    top_row(top, lo, hi, n, p.top, [&](int i) { return keys[i - lo]; }, [&](int at, int i) { out[at] = i; });
}

// ---- choosing tokens ----------------------------------------------------------------------------------
struct KeepParams {
    const float* w; int64_t w_rs;
    int Hkv, slots, keep, sinks, recent, cached;
    const int32_t* seq_lens;
    int32_t* kept; float* kept_w;
};

// order of the weights as unsigned numbers; NaN lowest, -0 as 0
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kTopThreads) tokens_select_kernel(KeepParams p) {
    extern __shared__ uint32_t ksm[];
    __shared__ TopShared top;
    cg::cluster_group cl = cg::this_cluster();
    const int bh = blockIdx.x / cl.num_blocks(), tid = threadIdx.x;
    const int n = min(max(p.seq_lens[bh / p.Hkv], 0), p.slots);
    const float* w = p.w + (int64_t)bh * p.w_rs;
    int lo, hi;
    top_slice(n, lo, hi);
    auto make = [&](int i) { return i < p.sinks || i >= n - p.recent ? 0xffffffffu : weight_key(__ldg(w + i)); };
    int32_t* kept = p.kept + (int64_t)bh * p.keep;
    float* kw = p.kept_w + (int64_t)bh * p.keep;
    for (int i = min(n, p.keep) + cl.block_rank() * kTopThreads + tid; i < p.keep; i += cl.num_blocks() * kTopThreads) {
        kept[i] = -1;
        kw[i] = 0.f;
    }
    auto put = [&](int at, int i) { kept[at] = i; kw[at] = __ldg(w + i); };
    if (p.cached) {
        for (int i = lo + tid; i < hi; i += kTopThreads) ksm[i - lo] = make(i);
        __syncthreads();
        top_row(top, lo, hi, n, p.keep, [&](int i) { return ksm[i - lo]; }, put);
    } else {
        top_row(top, lo, hi, n, p.keep, make, put);
    }
}

// ---- launches -------------------------------------------------------------------------------------------
// CTAs per row: enough rows x CTAs for the SMs, slices of 2048 keys or more, and small enough to be held.
static int top_cluster(int64_t rows, int64_t n, int sms, int64_t cap) {
    int c = 1;
    while (c < 8 && ((rows * c < sms && n / (2 * c) >= 2048) || (n + c - 1) / c > cap)) c *= 2;
    return c;
}

template <class K, class P>
static int launch_cluster(K kernel, const P& p, int64_t rows, int c, size_t smem, cudaStream_t st) {
    if (rows * c > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return PKV_ERR_CUDA;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * c));
    cfg.blockDim = dim3(kTopThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = c;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? PKV_OK : PKV_ERR_CUDA;
}

constexpr int64_t kKeyCap = 48 * 1024;          // keys of a slice in shared memory (192 KB)

int launch_tokens_select(const float* w, int B, int Hkv, int slots, int64_t rs, const int32_t* lens, int keep, int sinks,
                         int recent, int32_t* kept, float* kept_w, int sms, cudaStream_t st) {
    KeepParams p{w, rs, Hkv, slots, keep, sinks, recent, 0, lens, kept, kept_w};
    const int64_t rows = (int64_t)B * Hkv;
    const int c = top_cluster(rows, slots, sms, kKeyCap);
    const int64_t per = ((int64_t)slots + c - 1) / c;
    p.cached = per <= kKeyCap;
    return launch_cluster(tokens_select_kernel, p, rows, c, p.cached ? (size_t)per * 4 : 0, st);
}

// Shared memory of the selection without its keys; keys of a slice take what is left of 200 KB.
int launch_pages_select(const pkv_codec* c, Pages pg, const void* q, int qdt, int q_heads, int64_t q_bs, int64_t q_hs,
                        const int32_t* lens, const int8_t* sums, int top, int sinks, int recent, int32_t* out, int sms,
                        cudaStream_t st) {
    SelectParams p{};
    p.pg = pg;
    p.q = q; p.qdt = qdt; p.q_bs = q_bs; p.q_hs = q_hs;
    p.G = q_heads / pg.Hkv;
    p.dim = c->dim;
    p.pitch = (c->dim + 15) / 16 * 16;
    p.R = c->R;
    p.seq_lens = lens;
    p.sums = sums;
    p.top = top; p.sinks = sinks; p.recent = recent;
    p.out = out;
    const int64_t fixed = (int64_t)p.G * p.dim * 8 + 2 * (int64_t)p.G * p.pitch;
    const int64_t cap = (200 * 1024 - fixed) / 4, rows = (int64_t)pg.B * pg.Hkv;
    const int cl = top_cluster(rows, pg.max_pages, sms, cap);
    const int64_t per = ((int64_t)pg.max_pages + cl - 1) / cl;
    if (per > cap) return PKV_ERR_UNSUPPORTED;
    return launch_cluster(pages_select_kernel, p, rows, cl, (size_t)(fixed + per * 4), st);
}

int launch_pages_summarize(const pkv_codec* c, Pages pg, int cb, const int32_t* lens, const int32_t* start,
                           const int16_t* gz, const int16_t* gxy, int8_t* out, int sms, cudaStream_t st) {
    SummaryParams p{pg, lens, start, gz, gxy, out, c->dim / 3, cb, (c->dim + 15) / 16 * 16,
                    c->bits_r + c->bits_theta, (1 << (c->bits_z + c->bits_r + c->bits_theta)) - 1};
    const int64_t warps = (int64_t)pg.B * pg.max_pages * pg.Hkv;
    const int64_t ctas = (warps + 7) / 8;
    if (ctas > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    pages_summarize_kernel<<<(unsigned)ctas, 256, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? PKV_OK : PKV_ERR_CUDA;
}

int launch_pages_store(Pages pg, uint8_t* dst, const uint8_t* codes, int bytes, int n, const int32_t* start,
                       const int32_t* counts, cudaStream_t st) {
    const int64_t threads = (int64_t)pg.B * pg.Hkv * n * 8, ctas = (threads + 255) / 256;
    if (ctas > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    pages_store_kernel<<<(unsigned)ctas, 256, 0, st>>>(pg, dst, codes, bytes, n, start, counts);
    return cudaGetLastError() == cudaSuccess ? PKV_OK : PKV_ERR_CUDA;
}

int launch_tokens_gather(Pages s, Pages d, uint8_t* dk, uint8_t* dv, int bytes, const int32_t* kept, int keep, int sms,
                         cudaStream_t st) {
    const int64_t total = (int64_t)s.B * s.Hkv * keep * ((bytes + 15) / 16);
    const int64_t ctas = (total + 255) / 256;
    tokens_gather_kernel<<<(unsigned)(ctas < (int64_t)sms * 16 ? ctas : (int64_t)sms * 16), 256, 0, st>>>(s, d, dk, dv, bytes,
                                                                                                     kept, keep);
    return cudaGetLastError() == cudaSuccess ? PKV_OK : PKV_ERR_CUDA;
}

}  // namespace pkv
