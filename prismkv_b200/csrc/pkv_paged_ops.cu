// pkv_paged_ops.cu -- the kernels around attention over a paged code cache: storing rows, page
// summaries, choosing pages, choosing tokens to keep, and moving them.

#include <algorithm>
#include <climits>
#include <type_traits>

#include <cooperative_groups.h>

#include "pkv_paged.cuh"

namespace pkv {
namespace cg = cooperative_groups;

// ---- copies of code rows ------------------------------------------------------------------------
// Piece i of a row of m codes = `bytes` bytes: 16 bytes, the last one short when bytes % 16 != 0 (rows start on
// 16-byte boundaries; what lies behind a row in its last 16 bytes is neither read nor written).
__device__ __forceinline__ uint4 load_piece(const uint8_t* row, int bytes, int i) {
    const int at = i * 16;
    if (at + 16 <= bytes) return __ldcs(reinterpret_cast<const uint4*>(row + at));
    uint32_t w[4] = {0, 0, 0, 0};
    #pragma unroll
    for (int x = 0; x < 15; ++x)
        if (at + x < bytes) w[x >> 2] |= (uint32_t)row[at + x] << (8 * (x & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_piece(uint8_t* row, int bytes, int i, uint4 v) {
    const int at = i * 16;
    if (at + 16 <= bytes) {
        *reinterpret_cast<uint4*>(row + at) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    #pragma unroll
    for (int x = 0; x < 15; ++x)
        if (at + x < bytes) row[at + x] = (uint8_t)(w[x >> 2] >> (8 * (x & 3)));
}

// Rows (b, hk, i) of contiguous codes into slots start[b] + i, eight threads a row.  Unit: what a thread copies at a
// time -- 16 bytes where rows are whole pieces of that, else a code.
template <class Unit>
__global__ void __launch_bounds__(256) pages_store_kernel(Pages g, uint8_t* dst, const uint8_t* codes, int bytes, int n,
                                                          const int32_t* start, const int32_t* counts) {
    cudaGridDependencySynchronize();
    const int64_t rows = (int64_t)g.B * g.Hkv * n;
    const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    if (row >= rows) return;
    const int i = (int)(row % n), hk = (int)(row / n % g.Hkv), b = (int)(row / n / g.Hkv);
    if (counts && i >= input(counts + b)) return;
    const int64_t t = (int64_t)input(start + b) + i;
    if (t < 0 || t >= ((int64_t)g.max_pages << g.ps_log2)) {
        flag_error(kErrPage);
        return;
    }
    const int page = page_of(g, b, (int)(t >> g.ps_log2));
    if (page < 0) return;
    Unit* d = reinterpret_cast<Unit*>(dst + slot_offset(g, page, hk, (int)(t & ((1 << g.ps_log2) - 1))));
    const Unit* s = reinterpret_cast<const Unit*>(codes + row * bytes);
    for (int x = threadIdx.x & 7; x < bytes / (int)sizeof(Unit); x += 8) d[x] = s[x];
}

// Slots kept[b, hk, i] of the source pages into slots i of the destination's, K and V.  A CTA takes kGatherRows
// x (256 / pieces) neighbouring rows of one (sequence, KV head), a thread the same 16-byte piece of kGatherRows
// of them: the three dependent steps (slot, pages, codes) of its rows overlap.  The copies' bytes bound it: 32 x 16384
// rows of 64 bytes, K and V, take 27 us, 4.9 TB/s read and written.
constexpr int kGatherRows = 2;
__global__ void __launch_bounds__(256) tokens_gather_kernel(Pages s, Pages d, uint8_t* dk, uint8_t* dv, int bytes,
                                                            const int32_t* kept, int keep, int chunks) {
    constexpr int U = kGatherRows;
    const int pieces = (bytes + 15) / 16, rows = 256 / pieces;
    const int r = threadIdx.x / pieces, pc = threadIdx.x - r * pieces;
    const int bh = blockIdx.x / chunks, i0 = (blockIdx.x - bh * chunks) * rows * U + r;
    const int b = bh / s.Hkv, hk = bh - b * s.Hkv;
    cudaGridDependencySynchronize();
    if (r >= rows) return;
    int t[U];
    int64_t so[U], to[U];
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = i0 + u * rows;
        t[u] = i < keep ? input(kept + (int64_t)bh * keep + i) : -1;
    }
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = i0 + u * rows;
        so[u] = to[u] = -1;
        if (t[u] < 0) continue;
        const int sp = page_of(s, b, t[u] >> s.ps_log2), dp = page_of(d, b, i >> d.ps_log2);
        if (sp < 0 || dp < 0) continue;
        so[u] = slot_offset(s, sp, hk, t[u] & ((1 << s.ps_log2) - 1));
        to[u] = slot_offset(d, dp, hk, i & ((1 << d.ps_log2) - 1));
    }
    uint4 k[U], v[U];
    #pragma unroll
    for (int u = 0; u < U; ++u)
        if (so[u] >= 0) {
            k[u] = load_piece(s.k + so[u], bytes, pc);
            v[u] = load_piece(s.v + so[u], bytes, pc);
        }
    #pragma unroll
    for (int u = 0; u < U; ++u)
        if (so[u] >= 0) {
            store_piece(dk + to[u], bytes, pc, k[u]);
            store_piece(dv + to[u], bytes, pc, v[u]);
        }
}

// ---- page summaries -------------------------------------------------------------------------------
// Per page, KV head and channel the least and greatest grid value of the page's tokens; a step is 128
// grid values, so the floor is a shift and the ceiling a shift of the value + 127.
// One warp per (page, KV head).  LPT lanes hold a token's row, one 4-byte word (two or four codes) each, so a
// load covers 32 / LPT tokens; a lane keeps, per code, the least and greatest (x, y) as packed 16-bit pairs and
// of z the least and greatest bin (grid values rise with the bin).  (x, y) come from shared memory: up to 256
// entries in 32 copies, one per lane, so that lookups never collide; more entries in one copy, with conflicts.
// Memory latency bounds it -- a warp waits for a page's codes before it asks for the next page's -- at 63 % of the issue
// slots (7 instructions a code and lane, and about 300 a page for the reduction, the stores and the loop): 268 MB of codes
// in pages of 32 tokens take 94 us.
struct SummaryParams {
    Pages pg;
    const int32_t *seq_lens, *start;
    const int16_t *grid_z, *grid_xy;
    int8_t* out;
    int m, pitch, bits_z, bits_flat, index_mask, entries, chunk, chunks;
};

template <int CB, int LPT, bool COPIES>
__global__ void __launch_bounds__(256) pages_summarize_kernel(SummaryParams p) {
    __shared__ __align__(16) uint32_t lut[COPIES ? 256 * 32 : 4096];   // (x, y) grid values
    __shared__ int gz[256];
    constexpr int CW = 4 / CB, TPL = 32 / LPT, U = 8;       // codes per word, tokens per load, loads in flight
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunk = blockIdx.x % p.chunks, bh = blockIdx.x / p.chunks, b = bh / p.pg.Hkv, hk = bh - b * p.pg.Hkv;
    cudaGridDependencySynchronize();
    const int L = clamp_len(p.pg, input(p.seq_lens + b)), ps = 1 << p.pg.ps_log2;
    const int start = p.start ? max(input(p.start + b), 0) : 0;
    const int j0 = (start >> p.pg.ps_log2) + chunk * p.chunk;
    const int j1 = min(j0 + p.chunk, (int)(((int64_t)L + ps - 1) >> p.pg.ps_log2));
    if (j0 >= j1 || start >= L) return;
    const uint32_t* xy = reinterpret_cast<const uint32_t*>(p.grid_xy);
    int next = j0 + warp < j1 ? page_of(p.pg, b, j0 + warp) : -1;
    for (int i = tid; i < 1 << p.bits_z; i += 256) gz[i] = input(p.grid_z + i);
    if constexpr (COPIES) {                                  // 16-byte pieces of four copies, spread over the banks
        for (int e = tid; e < p.entries; e += 256) {
            const uint32_t v = input(xy + e);
            #pragma unroll
            for (int k = 0; k < 8; ++k) reinterpret_cast<uint4*>(lut)[e * 8 + ((k + e) & 7)] = make_uint4(v, v, v, v);
        }
    } else {
        for (int i = tid; i < p.entries; i += 256) lut[i] = input(xy + i);
    }
    __syncthreads();
    const int word = lane % LPT, tok = lane / LPT;
    const bool have = word * 4 < p.m * CB;                   // this lane's word holds codes of the row
    // byte address of a lookup: the index on the table's pitch (128 bytes of copies, or 4), plus the lane's copy
    constexpr int SH = COPIES ? 7 : 2;
    const uint32_t imask = (uint32_t)p.index_mask << SH, lane4 = COPIES ? lane * 4 : 0;
    const uint32_t zm = (1u << p.bits_z) - 1u, zmask = CB == 2 ? zm * 0x00010001u : zm * 0x01010101u;
    const char* const lutb = reinterpret_cast<const char*>(lut);
    const uint8_t* const mine = p.pg.k + (int64_t)hk * p.pg.head_bs + (int64_t)tok * p.pg.tok_bs + word * 4;
    for (int j = j0 + warp; j < j1; j += 8) {
        const int page = next;
        if (j + 8 < j1) next = page_of(p.pg, b, j + 8);
        if (page < 0) continue;
        const int n = min(L - (j << p.pg.ps_log2), ps);
        const uint8_t* row = mine + (int64_t)page * p.pg.page_bs;
        const int64_t step = TPL * p.pg.tok_bs;
        uint32_t lo[CW], hi[CW], zl[CW / 2], zh[CW / 2];     // z bins: two codes to a word
        #pragma unroll
        for (int x = 0; x < CW; ++x) { lo[x] = 0x7fff7fffu; hi[x] = 0x80008000u; }
        #pragma unroll
        for (int x = 0; x < CW / 2; ++x) { zl[x] = 0xffffffffu; zh[x] = 0u; }
        auto take = [&](uint32_t w) {
            #pragma unroll
            for (int x = 0; x < CW; ++x) {
                const int at = 8 * CB * x - SH;              // the code's lowest bit comes to bit SH
                const uint32_t a = (at < 0 ? w << -at : w >> at) & imask;
                const uint32_t v = *reinterpret_cast<const uint32_t*>(lutb + (a | lane4));
                lo[x] = __vmins2(lo[x], v);
                hi[x] = __vmaxs2(hi[x], v);
            }
            const uint32_t z = (w >> p.bits_flat) & zmask;
            #pragma unroll
            for (int x = 0; x < CW / 2; ++x) {               // CB 1: codes 0, 2 and codes 1, 3
                const uint32_t y = CB == 2 ? z : (z >> (8 * x)) & 0x00ff00ffu;
                zl[x] = __vminu2(zl[x], y);
                zh[x] = __vmaxu2(zh[x], y);
            }
        };
        if (have) {
            int r0 = 0;
            for (; r0 + U * TPL <= n; r0 += U * TPL) {       // U loads of whole groups of tokens in flight
                uint32_t w[U];
                #pragma unroll
                for (int u = 0; u < U; ++u) w[u] = __ldcs(reinterpret_cast<const uint32_t*>(row + u * step));
                row += U * step;
                #pragma unroll
                for (int u = 0; u < U; ++u) take(w[u]);
            }
            for (r0 += tok; r0 < n; r0 += TPL, row += step) take(__ldcs(reinterpret_cast<const uint32_t*>(row)));
        }
        #pragma unroll
        for (int off = LPT; off < 32; off <<= 1)
            #pragma unroll
            for (int x = 0; x < CW; ++x) {
                lo[x] = __vmins2(lo[x], __shfl_xor_sync(0xffffffffu, lo[x], off));
                hi[x] = __vmaxs2(hi[x], __shfl_xor_sync(0xffffffffu, hi[x], off));
                if (x < CW / 2) {
                    zl[x] = __vminu2(zl[x], __shfl_xor_sync(0xffffffffu, zl[x], off));
                    zh[x] = __vmaxu2(zh[x], __shfl_xor_sync(0xffffffffu, zh[x], off));
                }
            }
        int8_t* o = p.out + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch;
        // lanes of the first token write the least, those of the next (or the same) the greatest: 3 CW bytes
        #pragma unroll
        for (int side = 0; side < 2; ++side) {
            if (!have || tok != (TPL > 1 ? side : 0)) continue;
            int8_t v[3 * CW];
            #pragma unroll
            for (int x = 0; x < CW; ++x) {
                // code x's bin: CB 2: half x; CB 1: half x / 2 of word x % 2
                const int zw = CB == 2 ? 0 : x & 1, zs = CB == 2 ? 16 * x : 16 * (x >> 1);
                const uint32_t xyv = side ? hi[x] : lo[x];
                const int up = side ? 127 : 0;
                v[3 * x] = (int8_t)((gz[((side ? zh[zw] : zl[zw]) >> zs) & 0xffu] + up) >> 7);
                v[3 * x + 1] = (int8_t)(((int16_t)xyv + up) >> 7);
                v[3 * x + 2] = (int8_t)(((int16_t)(xyv >> 16) + up) >> 7);
            }
            int8_t* d = o + side * p.pitch + 3 * CW * word;
            if ((word + 1) * CW <= p.m) {
                using Out = typename std::conditional<CB == 2, uint16_t, uint32_t>::type;   // 3 CW bytes as three
                #pragma unroll
                for (int y = 0; y < 3; ++y) {
                    Out t = 0;
                    #pragma unroll
                    for (int z = 0; z < (int)sizeof(Out); ++z) t |= (Out)((Out)(uint8_t)v[y * (int)sizeof(Out) + z] << (8 * z));
                    reinterpret_cast<Out*>(d)[y] = t;
                }
            } else {                                         // the row's last word, not full
                #pragma unroll
                for (int y = 0; y < 3 * CW; ++y)
                    if (word * CW + y / 3 < p.m) d[y] = v[y];
            }
        }
        for (int d = 3 * p.m + lane; d < p.pitch; d += 32) o[d] = o[p.pitch + d] = 0;
    }
}

// ---- the k largest of a row, in index order ---------------------------------------------------------
// A cluster of CTAs holds a row of n keys (unsigned, larger = better): CTA `rank` the slice [lo, hi), its
// warps contiguous parts of that.  Histograms of the key's digits from the top narrow the k-th largest key;
// then every warp counts the keys of its part above and equal to it, and writes their indexes behind those of
// the parts before it (of the equal ones the first `need` of the row).  One cluster barrier per digit: every CTA
// sums all CTAs' histograms for itself, and the histograms of two digits alternate.
// What bounds it: a handful of barriers and round trips through the cluster's shared memory for short rows, the
// passes over the keys in shared memory for long ones.
template <int THREADS, int DIGIT>
struct TopShared {
    alignas(16) uint32_t hist[2][1 << DIGIT];
    uint32_t warp[2][THREADS / 32];
    uint32_t total[2];                         // this CTA's keys above and equal to the threshold
    uint32_t bin, need;
};

// BITS-bit keys in digits of DIGIT bits (the last one may be shorter).  put(at, x, i): key i, which is x, goes to
// place at.
template <int BITS, int THREADS, int DIGIT, class Key, class Put>
__device__ void top_row(TopShared<THREADS, DIGIT>& s, int lo, int hi, int n, int k, Key key, Put put) {
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rank = cl.block_rank(), C = cl.num_blocks();
    constexpr int BINS = 1 << DIGIT, PER = BINS > THREADS ? 2 : 1, PASSES = (BITS + DIGIT - 1) / DIGIT;
    static_assert(BINS <= 2 * THREADS, "bins per thread");
    uint32_t prefix = 0, need = (uint32_t)min(k, n);        // keys still to take among those with this prefix
    const bool all = n <= k;
    for (int i = tid; i < 2 * BINS; i += THREADS) (&s.hist[0][0])[i] = 0;
    __syncthreads();
    if (!all) {
        int shift = BITS;
        #pragma unroll 1
        for (int pass = 0; pass < PASSES; ++pass) {
            const int bits = min(DIGIT, shift), low = shift - bits;
            uint32_t* hist = s.hist[pass & 1];
            const uint32_t field = (1u << bits) - 1u, want = shift < 32 ? prefix >> shift : 0u;
            auto note = [&](uint32_t x) {
                if (shift == BITS || (x >> shift) == want) atomicAdd(&hist[(x >> low) & field], 1u);
            };
            int i = lo + tid;
            for (; i + 3 * THREADS < hi; i += 4 * THREADS) {
                const uint32_t x0 = key(i), x1 = key(i + THREADS), x2 = key(i + 2 * THREADS), x3 = key(i + 3 * THREADS);
                note(x0); note(x1); note(x2); note(x3);
            }
            for (; i < hi; i += THREADS) note(key(i));
            cl.sync();
            if (pass + 2 < PASSES + 1 && pass > 0)          // the other one was read before this barrier
                for (int i = tid; i < BINS; i += THREADS) s.hist[(pass + 1) & 1][i] = 0;
            // bins from the top, PER neighbouring ones a thread, summed over the cluster
            uint32_t v[PER], sum = 0;
            #pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = 0;
            if (PER * tid < BINS) {
                #pragma unroll 4
                for (unsigned r = 0; r < C; ++r) {
                    const uint32_t* h = cl.map_shared_rank(&s, r)->hist[pass & 1];
                    if constexpr (PER == 2) {
                        const uint2 x = reinterpret_cast<const uint2*>(h)[BINS / 2 - 1 - tid];
                        v[0] += x.y; v[1] += x.x;
                    } else {
                        v[0] += h[BINS - 1 - tid];
                    }
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
            #pragma unroll
            for (int w = 0; w < (THREADS / 32); ++w) inc += w < warp ? s.warp[0][w] : 0u;
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
    const int part = (hi - lo + (THREADS / 32) - 1) / (THREADS / 32);
    const int w0 = min(hi, lo + warp * part), w1 = min(hi, w0 + part);
    uint32_t above = 0, equal = 0;
    {
        auto note = [&](uint32_t x) {
            above += x > prefix;
            equal += x == prefix;
        };
        int i = w0 + lane;
        if (all) {
            above = i < w1 ? (uint32_t)(w1 - i + 31) / 32 : 0u;
        } else {
            for (; i + 96 < w1; i += 128) {
                const uint32_t x0 = key(i), x1 = key(i + 32), x2 = key(i + 64), x3 = key(i + 96);
                note(x0); note(x1); note(x2); note(x3);
            }
            for (; i < w1; i += 32) note(key(i));
        }
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) { s.warp[0][warp] = above; s.warp[1][warp] = equal; }
    __syncthreads();
    uint32_t pa = 0, pe = 0, ta = 0, te = 0;
    for (int w = 0; w < (THREADS / 32); ++w) {
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
    pa += min(pe, need);                                     // places before this part
    const unsigned below = (1u << lane) - 1u;
    for (int i0 = w0; i0 < w1; i0 += 128) {                  // four neighbouring keys a lane
        const int i = i0 + 4 * lane;
        uint32_t take = 0, same = 0;                         // keys above the threshold, and equal to it
        #pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t x = i + u < w1 ? key(i + u) : 0u;
            take |= (uint32_t)(i + u < w1 && (all || x > prefix)) << u;
            same |= (uint32_t)(i + u < w1 && !all && x == prefix) << u;
        }
        if (__any_sync(0xffffffffu, same)) {                 // of the equal ones the first `need` of the row
            const uint32_t ce = __popc(same);
            const unsigned e0 = __ballot_sync(0xffffffffu, ce & 1), e1 = __ballot_sync(0xffffffffu, ce & 2),
                           e2 = __ballot_sync(0xffffffffu, ce & 4);
            uint32_t ea = pe + __popc(e0 & below) + 2 * __popc(e1 & below) + 4 * __popc(e2 & below);
            pe += __popc(e0) + 2 * __popc(e1) + 4 * __popc(e2);
            for (; same; same &= same - 1, ++ea)
                if (ea < need) take |= same & (0u - same);
        }
        // places: counts (0 to 4) of the lanes below, bit by bit
        const uint32_t ca = __popc(take);
        const unsigned a0 = __ballot_sync(0xffffffffu, ca & 1), a1 = __ballot_sync(0xffffffffu, ca & 2),
                       a2 = __ballot_sync(0xffffffffu, ca & 4);
        uint32_t at = pa + __popc(a0 & below) + 2 * __popc(a1 & below) + 4 * __popc(a2 & below);
        pa += __popc(a0) + 2 * __popc(a1) + 4 * __popc(a2);
        for (; take; take &= take - 1, ++at) {               // (few lanes have more than one)
            const int k = i + __ffs(take) - 1;
            put((int)at, key(k), k);
        }
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
//    for long sequences; they are asked into L2 before the rotation starts.  32 rows of 4096 pages take 25 us: rotation
//    3, scores 7, digits 6, the rest latencies of the start, the order and the barriers.
//  * A score is below 192 * 127 * 127 < 2^22 in magnitude: keys of 24 bits, three digits of 8 (a digit costs about
//    2 us of barriers and remote reads with 256 bins, 5 us with 4096).
constexpr int kPageDigit = 8;
constexpr int kPageThreads = 512, kPageWarps = kPageThreads / 32;
constexpr uint32_t kForcedKey = 0xffffffu;

// PPL: 16-byte pieces of a summary per lane, at most
template <int PPL>
__global__ void __launch_bounds__(kPageThreads) pages_select_kernel(SelectParams p) {
    constexpr int U = PPL <= 3 ? 4 : 2;                      // pages a lane group has in flight
    extern __shared__ __align__(16) uint8_t ssm[];
    __shared__ TopShared<kPageThreads, kPageDigit> top;
    __shared__ double amax_w[kPageWarps];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, dim = p.dim;
    const int rank = cl.block_rank(), C = cl.num_blocks();
    const int bh = blockIdx.x / C, b = bh / p.pg.Hkv, hk = bh % p.pg.Hkv;
    cudaGridDependencySynchronize();
    const int L = clamp_len(p.pg, input(p.seq_lens + b));
    const int n = (int)(((int64_t)L + (1 << p.pg.ps_log2) - 1) >> p.pg.ps_log2);
    int8_t* qp = reinterpret_cast<int8_t*>(ssm);                       // [G][2][pitch] negative, then positive parts
    double* sq = reinterpret_cast<double*>(qp + 2 * p.G * p.pitch);    // [G][dim] (pitch: a multiple of 16)
    float* raw = reinterpret_cast<float*>(sq + p.G * dim);             // [G][dim]
    uint32_t* keys = reinterpret_cast<uint32_t*>(raw + p.G * dim);
    int lo, hi;
    top_slice(n, lo, hi);
    for (int i = tid; i < p.G * dim; i += kPageThreads)
        raw[i] = load_any(p.q, p.qdt, b * p.q_bs + (int64_t)(hk * p.G + i / dim) * p.q_hs + i % dim);
    for (int j = lo + tid; j < hi; j += kPageThreads)
        if (j >= p.sinks && j < n - p.recent) {
            const int page = page_of(p.pg, b, j);
            if (page >= 0)
                for (int x = 0; x < 2 * p.pitch; x += 64)       // (64 apart: a summary need not start a line)
                    prefetch_l2(p.sums + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch + x);
        }
    cl.sync();                                               // raw queries; every CTA of the cluster runs
    for (int k = rank * kPageWarps + warp; k < dim; k += C * kPageWarps) {
        float r[6];
        #pragma unroll
        for (int x = 0; x < 6; ++x) r[x] = lane + 32 * x < dim ? input(p.R + k * dim + lane + 32 * x) : 0.f;
        for (int h0 = 0; h0 < p.G; h0 += 4) {
            double a[4] = {0.0, 0.0, 0.0, 0.0};
            #pragma unroll
            for (int x = 0; x < 6; ++x)
                if (32 * x < dim && lane + 32 * x < dim) {
                    #pragma unroll
                    for (int h = 0; h < 4; ++h)
                        if (h0 + h < p.G) a[h] = fma((double)raw[(h0 + h) * dim + lane + 32 * x], (double)r[x], a[h]);
                }
            // four sums over the warp: half the lanes keep two heads, a quarter one, then a butterfly over eight
            const bool up16 = lane & 16, up8 = lane & 8;
            const double b0 = (up16 ? a[2] : a[0]) + __shfl_xor_sync(0xffffffffu, up16 ? a[0] : a[2], 16);
            const double b1 = (up16 ? a[3] : a[1]) + __shfl_xor_sync(0xffffffffu, up16 ? a[1] : a[3], 16);
            double v = (up8 ? b1 : b0) + __shfl_xor_sync(0xffffffffu, up8 ? b0 : b1, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            const int h = h0 + (lane >> 3);
            if ((lane & 7) < C && h < p.G) cl.map_shared_rank(sq, lane & 7)[h * dim + k] = v;
        }
    }
    cl.sync();
    double amax = 0.0;
    for (int i = tid; i < p.G * dim; i += kPageThreads) {
        const double a = fabs(sq[i]);
        amax = a <= 1e300 ? fmax(amax, a) : INFINITY;       // NaN too
        if (amax == INFINITY) break;
    }
    #pragma unroll
    for (int off = 16; off >= 1; off >>= 1) amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (lane == 0) amax_w[warp] = amax;
    __syncthreads();
    amax = 0.0;
    for (int w = 0; w < kPageWarps; ++w) amax = fmax(amax, amax_w[w]);
    for (int i = tid; i < p.G * p.pitch; i += kPageThreads) {
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
    for (int j0 = lo + warp * 32; j0 < hi; j0 += kPageWarps * 32) {
        // a lane finds one page; then eight groups of four lanes score U of the 32 pages at a time
        int mine = -1;
        {
            const int j = j0 + lane;
            if (j < hi && j >= p.sinks && j < n - p.recent) mine = page_of(p.pg, b, j);
        }
        #pragma unroll 1
        for (int u0 = 0; u0 < 4 && j0 + 8 * u0 < hi; u0 += U) {
            int4 w[U][PPL];
            #pragma unroll
            for (int u = 0; u < U; ++u) {
                const int page = __shfl_sync(0xffffffffu, mine, 8 * (u0 + u) + (lane >> 2));
                const int4* sum = reinterpret_cast<const int4*>(p.sums + ((int64_t)page * p.pg.Hkv + hk) * 2 * p.pitch) + sub;
                #pragma unroll
                for (int x = 0; x < PPL; ++x) {
                    w[u][x] = make_int4(0, 0, 0, 0);
                    if (page >= 0 && sub + 4 * x < pieces) w[u][x] = __ldcs(sum + 4 * x);
                }
            }
            int best[U];
            #pragma unroll
            for (int u = 0; u < U; ++u) best[u] = INT_MIN;
            #pragma unroll 2
            for (int h = 0; h < p.G; ++h) {
                int a[U] = {};
                #pragma unroll
                for (int x = 0; x < PPL; ++x)
                    if (sub + 4 * x < pieces) {
                        const int4 qv = q4[h * pieces + sub + 4 * x];
                        #pragma unroll
                        for (int u = 0; u < U; ++u) {
                            a[u] = __dp4a(w[u][x].x, qv.x, a[u]);
                            a[u] = __dp4a(w[u][x].y, qv.y, a[u]);
                            a[u] = __dp4a(w[u][x].z, qv.z, a[u]);
                            a[u] = __dp4a(w[u][x].w, qv.w, a[u]);
                        }
                    }
                #pragma unroll
                for (int u = 0; u < U; ++u) {
                    a[u] += __shfl_xor_sync(0xffffffffu, a[u], 1);
                    a[u] += __shfl_xor_sync(0xffffffffu, a[u], 2);
                    best[u] = max(best[u], a[u]);
                }
            }
            #pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + 8 * (u0 + u) + (lane >> 2);
                const int page = __shfl_sync(0xffffffffu, mine, 8 * (u0 + u) + (lane >> 2));
                if (sub == 0 && j < hi)
                    keys[j - lo] = j < p.sinks || j >= n - p.recent ? kForcedKey : page < 0 ? 0u : (uint32_t)(best[u] + (1 << 22));
            }
        }
    }
    __syncthreads();
    int32_t* out = p.out + (int64_t)bh * p.top;
    for (int i = min(n, p.top) + rank * kPageThreads + tid; i < p.top; i += C * kPageThreads) out[i] = -1;
    top_row<24, kPageThreads, kPageDigit>(top, lo, hi, n, p.top, [&](int i) { return keys[i - lo]; },
                              [&](int at, uint32_t, int i) { out[at] = i; });
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

// the weight of a key; keys of NaN, of either zero and of forced tokens do not tell theirs
__device__ __forceinline__ bool key_tells(uint32_t k) { return k != 0u && k != 0x80000000u && k != 0xffffffffu; }
__device__ __forceinline__ float key_weight(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// One cluster per (sequence, KV head).  The slice's keys lie in shared memory, computed once (a weight is read
// back from its key); where a slice does not fit they are computed from the weights on every pass.  Two sizes:
// 1024 threads and digits of 11 bits for long slices (3 passes over the keys), 512 threads and digits of 8 bits
// (4 passes, but 256 counters to clear, read and scan) up to kShortSlice keys: 8 rows of 1024 take 8 us, not 14.
// 32 rows of 131072 take 31 us, bound by the instructions of the passes over the keys.
constexpr int kShortSlice = 4096;

template <int THREADS, int DIGIT>
__global__ void __launch_bounds__(THREADS) tokens_select_kernel(KeepParams p) {
    extern __shared__ uint32_t ksm[];
    __shared__ TopShared<THREADS, DIGIT> top;
    cg::cluster_group cl = cg::this_cluster();
    const int bh = blockIdx.x / cl.num_blocks(), tid = threadIdx.x;
    cudaGridDependencySynchronize();
    const int n = min(max(input(p.seq_lens + bh / p.Hkv), 0), p.slots);
    const float* w = p.w + (int64_t)bh * p.w_rs;
    int lo, hi;
    top_slice(n, lo, hi);
    auto make = [&](int i, float x) { return i < p.sinks || i >= n - p.recent ? 0xffffffffu : weight_key(x); };
    int32_t* kept = p.kept + (int64_t)bh * p.keep;
    float* kw = p.kept_w + (int64_t)bh * p.keep;
    for (int i = min(n, p.keep) + cl.block_rank() * THREADS + tid; i < p.keep; i += cl.num_blocks() * THREADS) {
        kept[i] = -1;
        kw[i] = 0.f;
    }
    auto put = [&](int at, uint32_t x, int i) {
        kept[at] = i;
        kw[at] = key_tells(x) ? key_weight(x) : input(w + i);
    };
    if (p.cached) {
        constexpr int U = 16;                                // 64 KB of weights in flight per CTA
        for (int i0 = lo + tid; i0 < hi; i0 += U * THREADS) {
            float x[U];
            #pragma unroll
            for (int u = 0; u < U; ++u) x[u] = i0 + u * THREADS < hi ? input(w + i0 + u * THREADS) : 0.f;
            #pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * THREADS < hi) ksm[i0 + u * THREADS - lo] = make(i0 + u * THREADS, x[u]);
        }
        __syncthreads();
        top_row<32, THREADS, DIGIT>(top, lo, hi, n, p.keep, [&](int i) { return ksm[i - lo]; }, put);
    } else {
        top_row<32, THREADS, DIGIT>(top, lo, hi, n, p.keep, [&](int i) { return make(i, input(w + i)); }, put);
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
static int launch_cluster(K kernel, const P& p, int64_t rows, int c, int threads, size_t smem, cudaStream_t st,
                          std::atomic<int> (&seen)[64]) {
    if (rows * c > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    const int rc = allow_smem(kernel, (int)smem, seen);
    if (rc) return rc;
    return launch_behind(kernel, (unsigned)(rows * c), threads, smem, c, st, p);
}

constexpr int64_t kKeyCap = 46 * 1024;          // keys of a slice in shared memory (184 KB, beside 17 KB of counters)

int launch_tokens_select(const float* w, int B, int Hkv, int slots, int64_t rs, const int32_t* lens, int keep, int sinks,
                         int recent, int32_t* kept, float* kept_w, int sms, cudaStream_t st) {
    KeepParams p{w, rs, Hkv, slots, keep, sinks, recent, 0, lens, kept, kept_w};
    const int64_t rows = (int64_t)B * Hkv;
    const int c = top_cluster(rows, slots, sms, kKeyCap, 2048);
    const int64_t per = ((int64_t)slots + c - 1) / c;
    p.cached = per <= kKeyCap;
    const size_t smem = p.cached ? (size_t)per * 4 : 0;
    static std::atomic<int> seen_short[64], seen_long[64];
    if (per <= kShortSlice) return launch_cluster(tokens_select_kernel<512, 8>, p, rows, c, 512, smem, st, seen_short);
    return launch_cluster(tokens_select_kernel<1024, 11>, p, rows, c, 1024, smem, st, seen_long);
}

// Shared memory of the selection without its keys; keys of a slice take what is left of 190 KB, so that a cluster of
// eight holds those of a row of 303104 pages (16 heads of size 192) and more.
static int64_t select_fixed(int dim, int G) { return (int64_t)G * dim * 12 + 2 * (int64_t)G * ((dim + 15) / 16 * 16); }
static int64_t select_cap(int dim, int G) { return (190 * 1024 - select_fixed(dim, G)) / 4; }
bool pages_select_fits(int dim, int G, int max_pages) { return ((int64_t)max_pages + 7) / 8 <= select_cap(dim, G); }

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
    const int64_t fixed = select_fixed(p.dim, p.G), cap = select_cap(p.dim, p.G), rows = (int64_t)pg.B * pg.Hkv;
    const int cl = top_cluster(rows, pg.max_pages, sms, cap, 32);
    const int64_t per = ((int64_t)pg.max_pages + cl - 1) / cl;   // at most cap: pages_select_fits
    static std::atomic<int> seen3[64], seen6[64];
    const size_t smem = (size_t)(fixed + per * 4);
    if (2 * p.pitch <= 16 * 4 * 3) return launch_cluster(pages_select_kernel<3>, p, rows, cl, kPageThreads, smem, st, seen3);
    return launch_cluster(pages_select_kernel<6>, p, rows, cl, kPageThreads, smem, st, seen6);
}

template <int CB, int LPT>
static int launch_summaries(const SummaryParams& p, cudaStream_t st) {
    const int64_t ctas = (int64_t)p.pg.B * p.pg.Hkv * p.chunks;
    if (ctas > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    if (p.entries <= 256) return launch_behind(pages_summarize_kernel<CB, LPT, true>, (unsigned)ctas, 256, 0, 0, st, p);
    return launch_behind(pages_summarize_kernel<CB, LPT, false>, (unsigned)ctas, 256, 0, 0, st, p);
}

int launch_pages_summarize(const pkv_codec* c, Pages pg, int cb, const int32_t* lens, const int32_t* start,
                           const int16_t* gz, const int16_t* gxy, int8_t* out, int sms, cudaStream_t st) {
    SummaryParams p{};
    p.pg = pg;
    p.seq_lens = lens; p.start = start;
    p.grid_z = gz; p.grid_xy = gxy;
    p.out = out;
    p.m = c->dim / 3;
    p.pitch = (c->dim + 15) / 16 * 16;
    p.bits_z = c->bits_z;
    p.bits_flat = c->bits_r + c->bits_theta;
    p.index_mask = (1 << (c->xy_per_z ? p.bits_z + p.bits_flat : p.bits_flat)) - 1;
    p.entries = p.index_mask + 1;
    // CTAs: one wave of six per SM (33 KB of tables each), or one per (sequence, KV head) where those are more
    const int64_t rows = (int64_t)pg.B * pg.Hkv, per = std::max<int64_t>(1, 6 * (int64_t)sms / rows);
    p.chunk = (int)std::max<int64_t>(8, (pg.max_pages + per - 1) / per);
    p.chunks = (pg.max_pages + p.chunk - 1) / p.chunk;
    const int words = (p.m * cb + 3) / 4;
    if (cb == 1) return words <= 8 ? launch_summaries<1, 8>(p, st) : launch_summaries<1, 16>(p, st);
    return words <= 16 ? launch_summaries<2, 16>(p, st) : launch_summaries<2, 32>(p, st);
}

int launch_pages_store(Pages pg, uint8_t* dst, const uint8_t* codes, int bytes, int code_bytes, int n, const int32_t* start,
                       const int32_t* counts, cudaStream_t st) {
    const int64_t threads = (int64_t)pg.B * pg.Hkv * n * 8, ctas = (threads + 255) / 256;
    if (ctas > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)ctas;
    if (bytes % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0)
        return launch_behind(pages_store_kernel<uint4>, grid, 256, 0, 0, st, pg, dst, codes, bytes, n, start, counts);
    if (code_bytes == 2) return launch_behind(pages_store_kernel<uint16_t>, grid, 256, 0, 0, st, pg, dst, codes, bytes, n, start, counts);
    return launch_behind(pages_store_kernel<uint8_t>, grid, 256, 0, 0, st, pg, dst, codes, bytes, n, start, counts);
}

int launch_tokens_gather(Pages s, Pages d, uint8_t* dk, uint8_t* dv, int bytes, const int32_t* kept, int keep,
                         cudaStream_t st) {
    const int rows = 256 / ((bytes + 15) / 16) * kGatherRows, chunks = (keep + rows - 1) / rows;
    const int64_t ctas = (int64_t)s.B * s.Hkv * chunks;
    if (ctas > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    return launch_behind(tokens_gather_kernel, (unsigned)ctas, 256, 0, 0, st, s, d, dk, dv, bytes, kept, keep, chunks);
}

}  // namespace pkv
