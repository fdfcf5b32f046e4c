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
// A cluster of CTAs holds a row of n keys (unsigned, larger = better): CTA `rank` the slice [lo, hi), its
// warps contiguous parts of that.  Histograms of the key's digits from the top narrow the k-th largest key;
// then every warp counts the keys of its part above and equal to it, and writes their indexes behind those of
// the parts before it (of the equal ones the first `need` of the row).  One cluster barrier per digit: every CTA
// sums all CTAs' histograms for itself, and the histograms of two digits alternate.
// What bounds it: a handful of barriers and round trips through the cluster's shared memory for short rows, the
// passes over the keys in shared memory for long ones.
constexpr int kTopThreads = 512;
constexpr int kTopWarps = kTopThreads / 32;

template <int DIGIT>
struct TopShared {
    alignas(16) uint32_t hist[2][1 << DIGIT];
    uint32_t warp[2][kTopWarps];
    uint32_t total[2];                         // this CTA's keys above and equal to the threshold
    uint32_t bin, need;
};

// BITS-bit keys in digits of DIGIT bits (the last one may be shorter).  put(at, i): keys i, i + 32, i + 64,
// i + 96 go to places at[0 .. 3] (negative: not taken).
template <int BITS, int DIGIT, class Key, class Put>
__device__ void top_row(TopShared<DIGIT>& s, int lo, int hi, int n, int k, Key key, Put put) {
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rank = cl.block_rank(), C = cl.num_blocks();
    constexpr int BINS = 1 << DIGIT, PER = BINS / kTopThreads, PASSES = (BITS + DIGIT - 1) / DIGIT;
    static_assert(PER % 4 == 0, "a thread's bins are read as 16-byte pieces");
    uint32_t prefix = 0, need = (uint32_t)min(k, n);        // keys still to take among those with this prefix
    const bool all = n <= k;
    for (int i = tid; i < 2 * BINS; i += kTopThreads) (&s.hist[0][0])[i] = 0;
    __syncthreads();
    if (!all) {
        int shift = BITS;
        #pragma unroll 1
        for (int pass = 0; pass < PASSES; ++pass) {
            const int bits = min(DIGIT, shift), low = shift - bits;
            uint32_t* hist = s.hist[pass & 1];
            for (int i0 = lo + tid; i0 < hi; i0 += 4 * kTopThreads) {
                uint32_t x[4];
                #pragma unroll
                for (int u = 0; u < 4; ++u) x[u] = i0 + u * kTopThreads < hi ? key(i0 + u * kTopThreads) : 0u;
                #pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (i0 + u * kTopThreads < hi && (shift == BITS || (x[u] >> shift) == (prefix >> shift)))
                        atomicAdd(&hist[(x[u] >> low) & ((1u << bits) - 1u)], 1u);
            }
            cl.sync();
            if (pass + 2 < PASSES + 1 && pass > 0)          // the other one was read before this barrier
                for (int i = tid; i < BINS; i += kTopThreads) s.hist[(pass + 1) & 1][i] = 0;
            // bins from the top, PER neighbouring ones a thread, summed over the cluster
            uint32_t v[PER], sum = 0;
            #pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = 0;
            #pragma unroll 2
            for (unsigned r = 0; r < C; ++r) {
                const uint4* h = reinterpret_cast<const uint4*>(cl.map_shared_rank(&s, r)->hist[pass & 1]);
                #pragma unroll
                for (int j = 0; j < PER; j += 4) {
                    const uint4 x = h[(BINS - 4 - (tid * PER + j)) / 4];
                    v[j] += x.w; v[j + 1] += x.z; v[j + 2] += x.y; v[j + 3] += x.x;
                }
            }
            #pragma unroll
            for (int j = 0; j < PER; ++j) sum += v[j];
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
            #pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (cum < need && cum + v[j] >= need) {
                    s.bin = BINS - 1 - (tid * PER + j);
                    s.need = need - cum;
                }
                cum += v[j];
            }
            __syncthreads();
            prefix |= s.bin << low;
            need = s.need;
            shift = low;
            __syncthreads();
        }
    }
    // this warp's part, and its keys above and equal to the threshold
    const int part = (hi - lo + kTopWarps - 1) / kTopWarps;
    const int w0 = min(hi, lo + warp * part), w1 = min(hi, w0 + part);
    uint32_t above = 0, equal = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t x = key(i);
        above += all || x > prefix;
        equal += !all && x == prefix;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) { s.warp[0][warp] = above; s.warp[1][warp] = equal; }
    __syncthreads();
    uint32_t pa = 0, pe = 0, ta = 0, te = 0;
    for (int w = 0; w < kTopWarps; ++w) {
        if (w == warp) { pa = ta; pe = te; }
        ta += s.warp[0][w];
        te += s.warp[1][w];
    }
    if (tid == 0) { s.total[0] = ta; s.total[1] = te; }
    cl.sync();
    for (unsigned r = 0; r < rank; ++r) {
        const uint32_t* t = cl.map_shared_rank(&s, r)->total;
        pa += t[0];
        pe += t[1];
    }
    const unsigned below = (1u << lane) - 1u;
    for (int i0 = w0; i0 < w1; i0 += 128) {
        int at[4];                                           // places of this lane's four keys, -1: not taken
        #pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + 32 * u + lane;
            const uint32_t x = i < w1 ? key(i) : 0u;
            const bool a = i < w1 && (all || x > prefix), e = i < w1 && !all && x == prefix;
            const unsigned ma = __ballot_sync(0xffffffffu, a), me = __ballot_sync(0xffffffffu, e);
            const uint32_t ea = pe + __popc(me & below);
            at[u] = a || (e && ea < need) ? (int)(pa + __popc(ma & below) + min(ea, need)) : -1;
            pa += __popc(ma);
            pe += __popc(me);
        }
        put(at, i0 + lane);
    }
    cl.sync();                                               // no CTA leaves while another reads its counts
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

// One cluster per (sequence, KV head), a slice of its pages per CTA.
//  * The queries are rotated in 64 bits -- a rounding to int8 must not turn on how a sum was ordered -- each CTA
//    a share of the rows of R for all heads, the results stored into every CTA's shared memory.
//  * Four lanes score a page: a summary is 2 pitch bytes in one piece, its 16-byte pieces go round the four
//    lanes, the int8 queries (positive parts against the greatest, negative ones against the least) lie in
//    shared memory in the same order, and __dp4a sums 32-bit integers exactly.  The summaries' bytes bound it
//    for long sequences; they are asked into L2 before the rotation starts.
//  * A score is below 192 * 127 * 127 < 2^22 in magnitude: keys of 24 bits, two digits of 12.
constexpr int kPageDigit = 12;
constexpr uint32_t kForcedKey = 0xffffffu;

__global__ void __launch_bounds__(kTopThreads) pages_select_kernel(SelectParams p) {
    extern __shared__ __align__(16) uint8_t ssm[];
    __shared__ TopShared<kPageDigit> top;
    __shared__ double amax_w[kTopWarps];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, dim = p.dim;
    const int rank = cl.block_rank(), C = cl.num_blocks();
    const int bh = blockIdx.x / C, b = bh / p.pg.Hkv, hk = bh % p.pg.Hkv;
    const int L = clamp_len(p.pg, p.seq_lens[b]);
    const int n = (int)(((int64_t)L + (1 << p.pg.ps_log2) - 1) >> p.pg.ps_log2);
    int8_t* qp = reinterpret_cast<int8_t*>(ssm);                       // [G][2][pitch] negative, then positive parts
    double* sq = reinterpret_cast<double*>(qp + 2 * p.G * p.pitch);    // [G][dim] (pitch: a multiple of 16)
    float* raw = reinterpret_cast<float*>(sq + p.G * dim);             // [G][dim]
    uint32_t* keys = reinterpret_cast<uint32_t*>(raw + p.G * dim);
    int lo, hi;
    top_slice(n, lo, hi);
    for (int i = tid; i < p.G * dim; i += kTopThreads)
        raw[i] = load_any(p.q, p.qdt, b * p.q_bs + (int64_t)(hk * p.G + i / dim) * p.q_hs + i % dim);
    for (int j = lo + tid; j < hi; j += kTopThreads)
        if (j >= p.sinks && j < n - p.recent) {
            const int page = page_of(p.pg, b, j);
            if (page >= 0)
                for (int x = 0; x < 2 * p.pitch; x += 64)       // (64 apart: a summary need not start a line)
                    prefetch_l2(p.sums + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch + x);
        }
    cl.sync();                                               // raw queries; every CTA of the cluster runs
    for (int k = rank * kTopWarps + warp; k < dim; k += C * kTopWarps) {
        float r[6];
        #pragma unroll
        for (int x = 0; x < 6; ++x) r[x] = lane + 32 * x < dim ? __ldg(p.R + k * dim + lane + 32 * x) : 0.f;
        for (int h = 0; h < p.G; ++h) {
            double a = 0.0;
            #pragma unroll
            for (int x = 0; x < 6; ++x)
                if (32 * x < dim && lane + 32 * x < dim) a = fma((double)raw[h * dim + lane + 32 * x], (double)r[x], a);
            #pragma unroll
            for (int off = 16; off >= 1; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
            if (lane < C) cl.map_shared_rank(sq, lane)[h * dim + k] = a;
        }
    }
    cl.sync();
    double amax = 0.0;
    for (int i = tid; i < p.G * dim; i += kTopThreads) {
        const double a = fabs(sq[i]);
        amax = a <= 1e300 ? fmax(amax, a) : INFINITY;       // NaN too
        if (amax == INFINITY) break;
    }
    #pragma unroll
    for (int off = 16; off >= 1; off >>= 1) amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (lane == 0) amax_w[warp] = amax;
    __syncthreads();
    amax = 0.0;
    for (int w = 0; w < kTopWarps; ++w) amax = fmax(amax, amax_w[w]);
    for (int i = tid; i < p.G * p.pitch; i += kTopThreads) {
        const int h = i / p.pitch, d = i % p.pitch;
        int v = 0;
        // a zero or non-finite group scores every page alike
        if (d < dim && amax > 0.0 && amax <= 1e300) v = (int)rint(sq[h * dim + d] * 127.0 / amax);
        qp[2 * h * p.pitch + d] = (int8_t)min(v, 0);
        qp[(2 * h + 1) * p.pitch + d] = (int8_t)max(v, 0);
    }
    __syncthreads();
    // ---- scores: four lanes a page, pieces lane & 3, + 4, ... -------------------------------------------
    const int pieces = 2 * p.pitch / 16, sub = lane & 3;
    const int4* q4 = reinterpret_cast<const int4*>(qp);
    for (int j0 = lo + warp * 8; j0 < hi; j0 += kTopWarps * 8) {
        const int j = j0 + (lane >> 2);
        const bool scored = j < hi && j >= p.sinks && j < n - p.recent;
        const int page = scored ? page_of(p.pg, b, j) : -1;
        int4 w[6];                                           // pitch <= 192: at most 24 pieces
        #pragma unroll
        for (int x = 0; x < 6; ++x) {
            w[x] = make_int4(0, 0, 0, 0);
            if (page >= 0 && sub + 4 * x < pieces)
                w[x] = __ldcs(reinterpret_cast<const int4*>(p.sums + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch) + sub + 4 * x);
        }
        int best = INT_MIN;
        for (int h = 0; h < p.G; ++h) {
            int a = 0;
            #pragma unroll
            for (int x = 0; x < 6; ++x)
                if (sub + 4 * x < pieces) {
                    const int4 qv = q4[h * pieces + sub + 4 * x];
                    a = __dp4a(w[x].x, qv.x, a);
                    a = __dp4a(w[x].y, qv.y, a);
                    a = __dp4a(w[x].z, qv.z, a);
                    a = __dp4a(w[x].w, qv.w, a);
                }
            a += __shfl_xor_sync(0xffffffffu, a, 1);
            a += __shfl_xor_sync(0xffffffffu, a, 2);
            best = max(best, a);
        }
        if (sub == 0 && j < hi) keys[j - lo] = !scored ? kForcedKey : page < 0 ? 0u : (uint32_t)(best + (1 << 22));
    }
    __syncthreads();
    int32_t* out = p.out + (int64_t)bh * p.top;
    for (int i = min(n, p.top) + rank * kTopThreads + tid; i < p.top; i += C * kTopThreads) out[i] = -1;
    top_row<24, kPageDigit>(top, lo, hi, n, p.top, [&](int i) { return keys[i - lo]; },
                              [&](const int (&at)[4], int i) {
                                  #pragma unroll
                                  for (int u = 0; u < 4; ++u)
                                      if (at[u] >= 0) out[at[u]] = i + 32 * u;
                              });
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
    __shared__ TopShared<11> top;
    cg::cluster_group cl = cg::this_cluster();
    const int bh = blockIdx.x / cl.num_blocks(), tid = threadIdx.x;
    const int n = min(max(p.seq_lens[bh / p.Hkv], 0), p.slots);
    const float* w = p.w + (int64_t)bh * p.w_rs;
    int lo, hi;
    top_slice(n, lo, hi);
    auto make = [&](int i, float x) { return i < p.sinks || i >= n - p.recent ? 0xffffffffu : weight_key(x); };
    int32_t* kept = p.kept + (int64_t)bh * p.keep;
    float* kw = p.kept_w + (int64_t)bh * p.keep;
    for (int i = min(n, p.keep) + cl.block_rank() * kTopThreads + tid; i < p.keep; i += cl.num_blocks() * kTopThreads) {
        kept[i] = -1;
        kw[i] = 0.f;
    }
    auto put = [&](const int (&at)[4], int i) {
        float x[4];
        #pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = at[u] >= 0 ? __ldg(w + i + 32 * u) : 0.f;
        #pragma unroll
        for (int u = 0; u < 4; ++u)
            if (at[u] >= 0) {
                kept[at[u]] = i + 32 * u;
                kw[at[u]] = x[u];
            }
    };
    if (p.cached) {
        #pragma unroll 8
        for (int i = lo + tid; i < hi; i += kTopThreads) ksm[i - lo] = make(i, __ldg(w + i));
        __syncthreads();
        top_row<32, 11>(top, lo, hi, n, p.keep, [&](int i) { return ksm[i - lo]; }, put);
    } else {
        top_row<32, 11>(top, lo, hi, n, p.keep, [&](int i) { return make(i, __ldg(w + i)); }, put);
    }
}

// ---- launches -------------------------------------------------------------------------------------------
// CTAs per row: as many as the SMs hold at once while slices keep `least` keys, more where slices must be held.
static int top_cluster(int64_t rows, int64_t n, int sms, int64_t cap, int64_t least) {
    int c = 1;
    while (c < 8 && ((rows * 2 * c <= sms && n / (2 * c) >= least) || (n + c - 1) / c > cap)) c *= 2;
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

constexpr int64_t kKeyCap = 48 * 1024;          // weights of a slice in shared memory (192 KB)

int launch_tokens_select(const float* w, int B, int Hkv, int slots, int64_t rs, const int32_t* lens, int keep, int sinks,
                         int recent, int32_t* kept, float* kept_w, int sms, cudaStream_t st) {
    KeepParams p{w, rs, Hkv, slots, keep, sinks, recent, 0, lens, kept, kept_w};
    const int64_t rows = (int64_t)B * Hkv;
    const int c = top_cluster(rows, slots, sms, kKeyCap, 2048);
    const int64_t per = ((int64_t)slots + c - 1) / c;
    p.cached = per <= kKeyCap;
    return launch_cluster(tokens_select_kernel, p, rows, c, p.cached ? (size_t)per * 4 : 0, st);
}

// Shared memory of the selection without its keys; keys of a slice take what is left of 190 KB.
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
    const int64_t fixed = (int64_t)p.G * p.dim * 12 + 2 * (int64_t)p.G * p.pitch;
    const int64_t cap = (190 * 1024 - fixed) / 4, rows = (int64_t)pg.B * pg.Hkv;
    const int cl = top_cluster(rows, pg.max_pages, sms, cap, 64);
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
