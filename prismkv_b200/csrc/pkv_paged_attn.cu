// pkv_paged_attn.cu -- decode attention of one token per sequence over a paged code cache.
//
//   out[b, h] = R^T ( sum_t p_t V^(t) / sum_t p_t ),   p_t = exp(scale (R q) . K^(t) - max)
//
// over the sequence's tokens or those of listed pages; optionally weights_out[t] = weights[t] +
// sum_h p_t / sum p.  Three launches, each started while the one before still runs (programmatic
// dependent launches; launch_behind says what each may read ahead of its grid dependency):
// paged_query_kernel rotates the queries into operand fragments, paged_attn_kernel leaves one partial
// state per (CTA, unit) range, paged_join_kernel joins a unit's ranges, normalises and rotates back (and,
// in further CTAs, adds the weights from the scores that the second launch kept).  Small calls are bound by
// the chain of memory round trips through the three (16 us for 37 tokens of 8 heads), large ones by the decode's
// dependent chain at four warps per scheduler (4 x 131072 tokens, 32 query over 8 KV heads, head size 96, two-byte codes:
// 163 us, 3.3 TB/s, half of the copy rate; 398 instructions per 16 tokens, issue slots 56 % used, shared-memory pipe 61 %,
// tensor pipe 22 %).

#include "pkv_paged.cuh"

namespace pkv {

constexpr int kHQ = 4;                         // query heads per block: with their hi and lo parts a tile's eight columns

// ---------------------------------------------------------------------------------------------
// paged_attn_kernel: both products on register-operand tensor-core tiles (mma.sync m16n8k16), the codes
// decoded straight into operand fragments by table lookups.
//
// Why not tcgen05: a unit's four heads are the narrow side of both products and the operands come out of a
// table lookup in registers; tcgen05 wants M >= 64 and operands in shared or tensor memory, and writing the
// decoded tiles there costs more shared-memory bandwidth than the lookups themselves.
//
// Numbers: every operand is an fp16 pair (hi, lo) equal to its fp32 value to 2^-22 (weights below 2^-15 of the running
// maximum's: to 2^-37 of that, half a step of a subnormal fp16 under the 2^12; one that rounds to zero still counts in
// the fp32 sum of the weights); sums are fp32.
//  * a decoded x, y (and z from a table) is a pair along the contraction: k-pair = (hi, lo);
//  * queries and softmax weights are pairs across the eight columns: column h < 4 is head h's hi part,
//    column h + 4 its lo part; both columns are added afterwards.  So all four cross products count.
//  * table values are scaled by a power of two that puts the largest in [2^9, 2^10), a bin width dz (MODE 0, 3) by
//    one that puts it in [1, 2), the queries per head -- z channels times that width -- by one that puts theirs in
//    [2^13, 2^14): pairs of normal fp16 whatever the ranges of the codec and the data.  Weights are 2^12 exp2(score - running max).
//  * MODE 0 (two-byte codes, 8 bits of (r, theta)) and 3 (one-byte codes), both with uniform z of up to 4 bits and
//    one polar grid: z = zc + (i - c) dz, c the middle bin, enters by its index -- for the scores as the exact fp16
//    subnormal i 2^-24 (EX: as i - c), for the values as the exact i - c; what does not depend on i is added outside.
//    Centred, because an uncentred sum of p i grows with every token and the tiles' sums truncate; dz is taken
//    over all bins, since neighbours' difference carries their rounding.
// Tables in shared memory: MODE 0, 3 and 1 (one-byte codes, any codec) hold 256 rows of 32 copies, copy `lane`
// for each lane: the 32 lookups of a warp never collide, and at a 64 KB-aligned address one byte permute of
// the code word makes a lookup's address (z: and a shift).  MODE 2 (two-byte codes of any codec) holds one copy of all 2^bits
// (x, y) -- 32 copies of 4096 do not fit -- and pays bank conflicts; a z table has 32 copies per bin.
//
// A warp takes a granule of NG times 16 tokens at a time; for 16 of them, lane = 4 g + c:
//  * scores: rows = tokens, k = triplets.  Lane (g, c) holds tokens rho(g), rho(g) + 8, rho(2 x) = x, rho(2 x + 1) =
//    (x ^ 1) + 4 (neighbouring rows of 64 bytes lie in different banks), and CPL triplets of each: 8c .. 8c + 7 of
//    the first 32, then its share of the rest.
//  * weights: two 8x8 transposes (movmatrix) turn the score tile into the B operand of p . v.
//  * values: rows = triplets, k = tokens.  Lane (g, c) holds tokens c, (c ^ 1) + 4 and both + 8, and CPL / 2
//    triplets of each: 4g .. 4g + 3 of the first 32, then its share of the rest.
// Codes come through shared memory, two iterations ahead: a warp's lane 0 brings its granules' rows of K and V by
// bulk copies into the warp's own two-stage ring and every warp waits on its own barriers alone, so no warp
// waits for another inside a range.  (Loaded into registers one iteration ahead instead, the codes cost
// spills and a quarter of the issue slots in waits: attend over 4 x 131072 tokens 184 us.)  A page is found
// through the range's page list in shared memory.  Every bit pattern decodes to something finite, so what lies
// behind a row or a sequence needs no clearing: its scores are masked and its weights zero.
// ---------------------------------------------------------------------------------------------
template <int MODE_, int CPL_, int NG_, int W_, int NB_, bool EX_>
struct PA {
    static constexpr int MODE = MODE_, CPL = CPL_, NG = NG_, W = W_, NB = NB_, HQ = kHQ * NB;
    static constexpr bool EX = EX_;
    static constexpr bool AFF = MODE == 0 || MODE == 3;     // z by its index
    static constexpr int CB = MODE & 1 ? 1 : 2;
    static constexpr int CPV = CPL / 2;                     // triplets per lane and token (values) = (x, y) m-tiles
    static constexpr int KW = CPL * CB / 4, VW = (CPV * CB + 3) / 4;
    static constexpr int RP = CPL * 4 * CB;                 // bytes of a code row in the ring, at most
    static constexpr int SLOT = NG * 16 * RP;               // a granule's rows of K, or of V
    static constexpr int UPPER = 4 * W * SLOT > 98304 ? 3 : 4;  // slots (K, V of two stages) above the tables
    static constexpr int CHUNK = 512;                        // pages of the list held at a time
    static constexpr int XY_BYTES = MODE == 2 ? 4096 * 8 : 256 * 32 * 8;
    static constexpr int Z_BYTES = AFF ? 0 : 256 * 32 * 4;
    static constexpr int THREADS = W * 32;
    static constexpr int NBZ = AFF ? CPL / 4 : CPL / 2;   // z steps of the scores
    static constexpr int FRAGS = 2 * (CPL + NBZ);           // query operand registers per lane
};

struct PASmem {                                             // offsets below the tables, in bytes
    int acc, wm, wl, red, next, bar, list, ring, end;
};
template <class T>
__host__ __device__ inline PASmem pa_smem(int dim) {
    PASmem s;
    s.acc = 0;                                              // [warps][HQ][dim]
    s.wm = s.acc + T::W * T::HQ * dim * 4;                  // [warps][HQ] max
    s.wl = s.wm + T::W * T::HQ * 4;                         // [warps][HQ] sum
    s.red = s.wl + T::W * T::HQ * 4;                          // [32] reduction
    s.next = s.red + 32 * 4;                                // the next range
    s.bar = (s.next + (int)sizeof(PagedItem) + 7) / 8 * 8;                   // [warps][2 stages]
    s.list = s.bar + T::W * 2 * 8;                          // [2][CHUNK] pages: this range's, the next one's
    s.ring = (s.list + 2 * T::CHUNK * 4 + 127) / 128 * 128; // slots UPPER .. 3
    s.end = s.ring + (4 - T::UPPER) * T::W * T::SLOT;
    return s;
}

// Uniform z bins: the middle bin c, its value and the bin width.
struct AffineZ { int c; float zc, dz; };
__device__ __forceinline__ AffineZ affine_z(const PagedParams& p) {
    const int n = 1 << p.bits_z, c = n >> 1;
    return {c, input(p.dec_z + c), (input(p.dec_z + n - 1) - input(p.dec_z)) / (float)(n - 1)};
}

// triplet j of lane c (scores), triplet i of lane g (values)
__device__ __forceinline__ int k_triplet_of(int cpl, int c, int j) {
    return j < 8 ? 8 * c + j : 32 + (cpl - 8) * c + (j - 8);
}
template <class T> __device__ __forceinline__ int v_triplet(int g, int i) {
    if (i < 4) return 4 * g + i;
    return 32 + (T::CPV - 4) * g + (i - 4);
}

// `BYTES` (2 to 16) of codes at a shared address into w[]
template <int BYTES> __device__ __forceinline__ void lds_codes(uint32_t* w, uint32_t at) {
    if constexpr (BYTES == 16) {
        const uint4 v = lds_u32x4(at);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (BYTES == 8) {
        const uint2 v = lds_u32x2m(at);
        w[0] = v.x; w[1] = v.y;
    } else if constexpr (BYTES == 4) {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
    } else {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
        w[0] = v;
    }
}

template <class T>
__device__ __forceinline__ void load_k(uint32_t (&w)[T::KW], uint32_t row, int c) {
    lds_codes<8 * T::CB>(w, row + 8 * T::CB * c);
    if constexpr (T::CPL > 8) lds_codes<(T::CPL - 8) * T::CB>(w + 8 * T::CB / 4, row + (32 + (T::CPL - 8) * c) * T::CB);
}
template <class T>
__device__ __forceinline__ void load_v(uint32_t (&w)[T::VW], uint32_t row, int g) {
    lds_codes<4 * T::CB>(w, row + 4 * T::CB * g);
    if constexpr (T::CPV > 4) lds_codes<(T::CPV - 4) * T::CB>(w + T::CB, row + (32 + (T::CPV - 4) * g) * T::CB);
}

// Lookups.  xy_reg / z_reg: the tables' shared addresses with the lane's copy in the low byte.
struct Lookup { uint32_t xy, z; int zsh; uint32_t zmask, xymask, mid; };   // mid: 1024 + c in both fp16 halves

template <class T> __device__ __forceinline__ uint2 look_xy(const Lookup& l, const uint32_t* w, int j) {
    if constexpr (T::MODE == 0) return lds_u32x2m(__byte_perm(w[j >> 1], l.xy, (j & 1) ? 0x7624u : 0x7604u));
    if constexpr (T::MODE & 1) return lds_u32x2m(__byte_perm(w[j >> 2], l.xy, 0x7604u + ((j & 3) << 4)));
    const uint32_t x = (j & 1) ? w[j >> 1] >> 13 : w[j >> 1] << 3;
    return lds_u32x2m((x & l.xymask) + l.xy);
}
// (z_hi, z_lo) from the table (MODE 1, 2)
template <class T> __device__ __forceinline__ uint32_t look_z(const Lookup& l, const uint32_t* w, int j) {
    uint32_t a, v;
    if constexpr (T::MODE == 1) {
        a = __byte_perm(w[j >> 2], l.z, 0x7604u + ((j & 3) << 4)) >> 1;   // rows of 128 bytes
    } else {
        const uint32_t code = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1];
        a = (((code >> l.zsh) & l.zmask) << 7) + l.z;
    }
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }
constexpr int kTabLim = 100, kQueryLim = 126;  // powers of two of tables and bin widths, and of queries, at most
// k with |v| 2^k in [2^top, 2^(top + 1)), held in [-lim, lim]; 0 for zero and non-finite v
__device__ __forceinline__ int pow2_to(float v, int top, int lim) {
    if (!(v > 0.f) || v > 3.402823466e38f) return 0;
    const int e = max((int)((__float_as_uint(v) >> 23) & 0xFF) - 127, -126);
    return max(-lim, min(lim, top - e));
}

// One CTA per block: q' = scale log2(e) R q of its four heads (zero for heads past the group), then the score
// operands of every lane, fragment r of lane l at frag[(block FRAGS + r) 32 + l]: pairs j < CPL of (x, y) of
// triplet j, then z; head h's power of two and the index-free part of its z sum at head[block 8 + h], + 4.
constexpr int kQueryThreads = 512;
__global__ void __launch_bounds__(kQueryThreads) paged_query_kernel(PagedParams p, int affine, int cpl, int ex) {
    extern __shared__ float qsm[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, dim = p.dim, unit = blockIdx.x;
    constexpr int NW = kQueryThreads / 32;
    float *sRaw = qsm, *sQ = qsm + kHQ * dim;
    __shared__ int sk[kHQ];
    const int per = p.UG * p.NB;                             // blocks per KV head
    const int b = unit / (p.pg.Hkv * per), u = unit % (p.pg.Hkv * per), hk = u / per, hg = u % per;
    // What the call reads is there from here on -- for the attention launch too, which comes up once every CTA of
    // this one is past this point, and reads pages and lengths before it waits for this one's results.
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const AffineZ az = affine_z(p);
    const float dz = az.dz * pow2(pow2_to(fabsf(az.dz), 0, kTabLim));
    float rr[6][6];                                          // rows warp, warp + NW, ... of R, six at a time
    auto load_rows = [&](int k0) {
        #pragma unroll
        for (int i = 0; i < 6; ++i)
            #pragma unroll
            for (int x = 0; x < 6; ++x) {
                const int k = k0 + i * NW, d = lane + 32 * x;
                rr[i][x] = (k < dim && d < dim) ? input(p.R + k * dim + d) : 0.f;
            }
    };
    load_rows(warp);
    for (int i = tid; i < kHQ * dim; i += kQueryThreads) {
        const int h = hg * kHQ + i / dim;
        sRaw[i] = h < p.G ? load_any(p.q, p.qdt, b * p.q_bs + (int64_t)(hk * p.G + h) * p.q_hs + i % dim) : 0.f;
    }
    __syncthreads();
    for (int k0 = warp; k0 < dim; k0 += 6 * NW) {
        if (k0 != warp) load_rows(k0);
        #pragma unroll
        for (int i = 0; i < 6; ++i) {
            const int k = k0 + i * NW;
            if (k >= dim) break;
            float a[kHQ] = {0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int x = 0; x < 6; ++x)
                if (32 * x < dim) {
                    const int d = min(lane + 32 * x, dim - 1);   // (rr is 0 behind the row)
                    #pragma unroll
                    for (int h = 0; h < kHQ; ++h) a[h] = fmaf(rr[i][x], sRaw[h * dim + d], a[h]);
                }
            // four sums over the warp: halve the lanes per head twice, then a butterfly over eight
            const bool up16 = lane & 16, up8 = lane & 8;
            const float b0 = (up16 ? a[2] : a[0]) + __shfl_xor_sync(0xffffffffu, up16 ? a[0] : a[2], 16);
            const float b1 = (up16 ? a[3] : a[1]) + __shfl_xor_sync(0xffffffffu, up16 ? a[1] : a[3], 16);
            float v = (up8 ? b1 : b0) + __shfl_xor_sync(0xffffffffu, up8 ? b0 : b1, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            if ((lane & 7) == 0) sQ[(lane >> 3) * dim + k] = v * p.scale_log2;
        }
    }
    __syncthreads();
    if (warp < kHQ) {
        float am = 0.f, cz = 0.f;
        for (int d = lane; d < dim; d += 32) {
            const float v = sQ[warp * dim + d];
            const bool isz = d % 3 == 0;
            am = fmaxf(am, fabsf(v) * (affine && isz ? fabsf(dz) : 1.f));
            if (isz) cz += v;
        }
        #pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, off));
            cz += __shfl_xor_sync(0xffffffffu, cz, off);
        }
        if (lane == 0) {
            const int k = pow2_to(am, 13, kQueryLim);
            sk[warp] = k;
            p.head[unit * 8 + warp] = __int_as_float(k);
            p.head[unit * 8 + 4 + warp] = affine ? cz * (ex ? az.zc : fmaf(-(float)az.c, az.dz, az.zc)) : 0.f;
        }
    }
    __syncthreads();
    const int nxy = 2 * cpl, frags = nxy + (affine ? cpl / 2 : cpl);
    const int g = lane >> 2, c = lane & 3, qh = g & 3;
    const bool lo = g >= 4;
    const float su = pow2(sk[qh]);
    auto qv = [&](int t, int x) { return t < p.m ? sQ[qh * dim + 3 * t + x] * su : 0.f; };
    for (int r = warp; r < frags; r += NW) {
        uint32_t v;
        if (r < nxy) {
            v = h2_dup_part(qv(k_triplet_of(cpl, c, r >> 1), 1 + (r & 1)), lo);
        } else if (affine) {                              // two triplets' z, times the scaled bin width
            const int j = 2 * (r - nxy);
            v = h2_pair_part(qv(k_triplet_of(cpl, c, j), 0) * dz, qv(k_triplet_of(cpl, c, j + 1), 0) * dz, lo);
        } else {
            v = h2_dup_part(qv(k_triplet_of(cpl, c, r - nxy), 0), lo);
        }
        p.frag[((int64_t)unit * frags + r) * 32 + lane] = v;
    }
}

// (i_a - c, i_b - c) as fp16 from the low nibbles of bytes 0 and 2
__device__ __forceinline__ uint32_t centred(uint32_t t, uint32_t mid) {
    const uint32_t h = (t & 0x000F000Fu) | 0x64006400u;      // 1024 + i, exact
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&mid));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// z by index, scores: the indexes of codes 4 j + 2 h, + 1 of a row's words, as the subnormals i 2^-24 or (EX: sums of
// q (i - c) are several times smaller, and so is what they lose) as i - c
template <class T> __device__ __forceinline__ uint32_t k_index(const Lookup& l, const uint32_t* w, int j, int h) {
    if constexpr (T::MODE == 0) {
        if constexpr (T::EX) return centred(w[2 * j + h] >> 8, l.mid);
        return prmt(w[2 * j + h], 0u, 0x4341u);
    } else {
        const uint32_t t = prmt((w[j] >> l.zsh) & l.zmask, 0u, h ? 0x4342u : 0x4140u);
        return T::EX ? centred(t, l.mid) : t;
    }
}
// values: i - c of triplet i's code for two tokens' words
template <class T> __device__ __forceinline__ uint32_t v_index(const Lookup& l, const uint32_t* wa, const uint32_t* wb, int i) {
    if constexpr (T::MODE == 0) return centred(prmt(wa[i >> 1], wb[i >> 1], (i & 1) ? 0x7733u : 0x5511u), l.mid);
    const int x = i & 3;
    return centred(prmt((wa[i >> 2] >> l.zsh) & l.zmask, (wb[i >> 2] >> l.zsh) & l.zmask,
                        (uint32_t)(x | x << 4 | (x + 4) << 8 | (x + 4) << 12)), l.mid);
}

// a . b on one tile, its sums started from zero
__device__ __forceinline__ void mma_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// d (+)= a . b (first: from zero); EX: the tile's sum joins d in a rounded fp32 addition (the tensor core truncates
// what it adds to d)
template <bool EX>
__device__ __forceinline__ void mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, bool first = false) {
    if (first) {
        mma_zero(d, a0, a1, a2, a3, b0, b1);
    } else if constexpr (EX) {
        float t[4];
        mma_zero(t, a0, a1, a2, a3, b0, b1);
        #pragma unroll
        for (int x = 0; x < 4; ++x) d[x] += t[x];
    } else {
        mma16816(d, a0, a1, a2, a3, b0, b1);
    }
}

template <class T>
__global__ void __launch_bounds__(T::THREADS, 1) paged_attn_kernel(PagedParams p) {
    extern __shared__ __align__(128) uint8_t pa_raw[];
    constexpr int W = T::W, NG = T::NG, CPL = T::CPL, CPV = T::CPV, MODE = T::MODE, nthr = T::THREADS;
    constexpr bool AFF = T::AFF;
    constexpr int NB = T::NB, HQ = T::HQ;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, dim = p.dim;
    cudaTriggerProgrammaticLaunchCompletion();
    const PASmem L = pa_smem<T>(dim);
    float *sAcc = reinterpret_cast<float*>(pa_raw + L.acc), *sRed = reinterpret_cast<float*>(pa_raw + L.red);
    float *sWm = reinterpret_cast<float*>(pa_raw + L.wm), *sWl = reinterpret_cast<float*>(pa_raw + L.wl);
    int* sList = reinterpret_cast<int*>(pa_raw + L.list);
    PagedItem* sNext = reinterpret_cast<PagedItem*>(pa_raw + L.next);
    uint64_t* bar = reinterpret_cast<uint64_t*>(pa_raw + L.bar) + warp * 2;
    // the tables start at the first 64 KB boundary of shared addresses behind the rest
    const uint32_t base = smem_u32(pa_raw);
    const uint32_t tab = (base + L.end + 0xFFFFu) & ~0xFFFFu;
    const uint32_t upper = tab + T::XY_BYTES + T::Z_BYTES;    // the ring's upper slots
    {
        uint32_t have;
        asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(have));
        if (upper + T::UPPER * W * T::SLOT + 128 > base + have) {   // the window lies elsewhere than planned for
            if (tid == 0) flag_error(kErrSmemLayout);
            cudaGridDependencySynchronize();
            return;
        }
    }
    uint8_t* tabp = pa_raw + (tab - base);
    if (lane == 0) {
        mbar_init(&bar[0], 1);
        mbar_init(&bar[1], 1);
        fence_mbar_init();
    }
    __syncwarp();

    // ---- tables: entries to registers, the largest magnitude, then the scaled pairs -----------------
    const int bits_all = p.bits_z + p.bits_flat;
    const AffineZ az = affine_z(p);                           // (AFF)
    constexpr int ENT = MODE == 2 ? 4096 : 256, EPT = (ENT + nthr - 1) / nthr;
    float2 exy[EPT];
    float ez[MODE == 1 ? EPT : 1];
    float am = 0.f;
    #pragma unroll
    for (int x = 0; x < EPT; ++x) {
        // codes past 2^bits (never stored by an encoder) read as code 0
        const int e = tid + x * nthr, code = e < (1 << bits_all) ? e : 0;
        exy[x] = __ldg(reinterpret_cast<const float2*>(p.dec_xy) +
                       (p.xy_per_z ? code : code & ((1 << p.bits_flat) - 1)));
        if (MODE == 1) ez[x] = __ldg(p.dec_z + (code >> p.bits_flat));
        am = fmaxf(am, fmaxf(fabsf(exy[x].x), fabsf(exy[x].y)));
    }
    if (!AFF)
        for (int i = tid; i < 1 << p.bits_z; i += nthr) am = fmaxf(am, fabsf(__ldg(p.dec_z + i)));
    PagedCursor cur = paged_begin(p);
    if (cur.t >= cur.end) {
        cudaGridDependencySynchronize();
        return;
    }
    int tk = 0;                                               // the tables' power of two (set below)
    auto fill_tables = [&] {
        const float ts = pow2(tk);
        #pragma unroll
        for (int x = 0; x < EPT; ++x) {
            const int e = tid + x * nthr;
            if (e >= ENT) break;
            if constexpr (MODE == 2)                          // (not held in registers: 16 of them)
                exy[x] = __ldg(reinterpret_cast<const float2*>(p.dec_xy) +
                               (p.xy_per_z ? e & ((1 << bits_all) - 1) : e & ((1 << p.bits_flat) - 1)));
            const uint2 v = make_uint2(h2_split(exy[x].x * ts), h2_split(exy[x].y * ts));
            if constexpr (MODE == 2) {
                reinterpret_cast<uint2*>(tabp)[e] = v;
            } else {
                // 32 copies in 16-byte pieces; a thread starts at its own piece, so that a warp's stores
                // spread over the banks (rows are 256 bytes apart)
                #pragma unroll
                for (int i = 0; i < 16; ++i)
                    reinterpret_cast<uint4*>(tabp)[e * 16 + ((i + tid) & 15)] = make_uint4(v.x, v.y, v.x, v.y);
                if constexpr (MODE == 1) {
                    const uint32_t z = h2_split(ez[x] * ts);
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        reinterpret_cast<uint4*>(tabp + T::XY_BYTES)[e * 8 + ((i + tid) & 7)] = make_uint4(z, z, z, z);
                }
            }
        }
        if constexpr (MODE == 2) {
            uint32_t* zt = reinterpret_cast<uint32_t*>(tabp + T::XY_BYTES);
            for (int i = tid; i < 32 << p.bits_z; i += nthr) zt[i] = h2_split(__ldg(p.dec_z + (i >> 5)) * ts);
        }
    };
    Lookup lk;
    lk.xy = MODE == 2 ? tab : tab | ((uint32_t)lane << 3);
    lk.z = MODE == 1 ? (tab + T::XY_BYTES) * 2 + ((uint32_t)lane << 3) : tab + T::XY_BYTES + ((uint32_t)lane << 2);
    lk.zsh = p.bits_flat;
    lk.mid = (0x6400u + (uint32_t)az.c) * 0x10001u;
    lk.zmask = ((1u << p.bits_z) - 1u) * (MODE == 3 ? 0x01010101u : 1u);
    lk.xymask = ((1u << bits_all) - 1u) << 3;

    const int g = lane >> 2, c = lane & 3, hp = c & 1;
    const int rho = ((g >> 1) ^ (g & 1)) + 4 * (g & 1);
    const int psl = p.pg.ps_log2, tokb = (int)p.pg.tok_bs;
    const int pitch = (p.m * T::CB + 15) & ~15;               // bytes of a row in the ring
    const bool whole = p.pg.tok_bs == pitch;                  // a granule's rows are one piece
    // Pages of granules [ga, gb) of an item as id, -1 (masked), or id | sign bit (the sequence's last page)
    PagedItem it{};
    int lbuf = 0;
    constexpr int GL = NG == 2 ? 5 : 4;                       // log2 of a granule's tokens (CHUNK is even)
    auto list_end = [&](const PagedItem& i, int ga) {
        return (int)min((int64_t)i.g1, ((int64_t)((ga << GL >> psl) + T::CHUNK) << psl) >> GL);
    };
    // pages that the item's sequence (or list) has
    auto page_end = [&](const PagedItem& i, int n) { return p.selected ? p.n_sel : (n + (1 << psl) - 1) >> psl; };
    auto list_load = [&](const PagedItem& i, int ga, int* list) {
        const int n = clamp_len(p.pg, input(p.seq_lens + i.b)), last = (n - 1) >> psl;
        const int j0 = ga << GL >> psl, j1 = ((list_end(i, ga) << GL) - 1) >> psl, je = page_end(i, n);
        for (int j = j0 + tid; j <= j1; j += nthr) {
            const RangePage r = j < je ? range_page(p, i.b, i.hk, j) : RangePage{-1, -1};
            list[j - j0] = r.page < 0 ? -1 : r.logical == last ? r.page | (int)0x80000000 : r.page;
        }
    };
    int gi = 0, ga = 0, gb = 0, lastn = 0;
    const uint8_t *kpool = nullptr, *vpool = nullptr;        // the item's KV head of page 0
    // The warp's slots of the stage in turn, and those of both added up: the other stage's are sum - mine.
    auto slot_at = [&](int x) {
        return x < T::UPPER ? upper + (uint32_t)(x * W + warp) * T::SLOT : base + (uint32_t)L.ring + (uint32_t)warp * T::SLOT;
    };
    uint32_t sk = slot_at(0), sv = slot_at(1);
    const uint32_t bothk = sk + slot_at(2), bothv = sv + slot_at(3);
    int stage = 0;
    uint32_t phase = 0;                                      // parities of the stages' next waits, one bit each
    bool ok = true;                                          // no wait ran out
    // Ask for granule x into the stage in turn (other: into the other one), whose last reads are done; tokens that
    // count in each of its sixteens, 8 bits apiece.
    auto ask = [&](int x, bool other) -> int {
        if (x >= gb || !ok) return 0;
        int n[NG], cnt = 0, have = 0;
        int64_t o[NG];
        #pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int t = (x << GL) + 16 * i, slot = t & ((1 << psl) - 1);
            const int e = sList[lbuf * T::CHUNK + (t >> psl) - (ga << GL >> psl)];
            n[i] = e == -1 ? 0 : e < 0 ? max(0, min(16, lastn - slot)) : 16;
            o[i] = (int64_t)(e & 0x7fffffff) * (int)p.pg.page_bs + slot * tokb;
            cnt |= n[i] << (8 * i);
            have += n[i] > 0;
        }
        if (have == 0) return 0;
        uint64_t* b = &bar[other ? stage ^ 1 : stage];
        const uint32_t dk = other ? bothk - sk : sk, dv = other ? bothv - sv : sv;
        const uint32_t bytes = (uint32_t)(16 * pitch);
        if (whole) {
            if (lane == 0) {
                mbar_arrive_expect_tx(b, 2 * have * bytes);
                if (NG == 2 && n[NG - 1] > 0 && o[NG - 1] == o[0] + (int)bytes) {   // 32 rows in one piece
                    bulk_g2s_at(dk, kpool + o[0], 2 * bytes, b);
                    bulk_g2s_at(dv, vpool + o[0], 2 * bytes, b);
                } else {
                    #pragma unroll
                    for (int i = 0; i < NG; ++i)
                        if (n[i] > 0) {
                            bulk_g2s_at(dk + i * bytes, kpool + o[i], bytes, b);
                            bulk_g2s_at(dv + i * bytes, vpool + o[i], bytes, b);
                        }
                }
            }
        } else {                                             // strided rows: one copy each, lane r for row r
            if (lane == 0) mbar_arrive_expect_tx(b, 2 * have * bytes);
            __syncwarp();
            if (lane < 16) {
                #pragma unroll
                for (int i = 0; i < NG; ++i)
                    if (n[i] > 0) {
                        const int64_t at = o[i] + lane * tokb;
                        bulk_g2s_at(dk + i * bytes + lane * pitch, kpool + at, (uint32_t)pitch, b);
                        bulk_g2s_at(dv + i * bytes + lane * pitch, vpool + at, (uint32_t)pitch, b);
                    }
            }
        }
        return cnt;
    };
    // the first granules of the list: warp w takes granules w, w + W, ...
    int cnt = 0, cnt2 = 0;                                   // of this iteration and the next one
    auto start_list = [&](int from) {
        ga = from;
        gb = list_end(it, ga);
        gi = ga + warp;
        cnt = ask(gi, false);
        cnt2 = ask(gi + W, true);
    };
    auto start_item = [&] {
        const int len = clamp_len(p.pg, input(p.seq_lens + it.b));
        lastn = len - ((len - 1) >> psl << psl);             // tokens of the sequence's last page
        kpool = p.pg.k + (int64_t)it.hk * p.pg.head_bs;
        vpool = p.pg.v + (int64_t)it.hk * p.pg.head_bs;
        start_list(it.g0);
    };
    uint32_t bq[NB][CPL][2], bz[NB][T::NBZ][2];
    // heads 2 hp, 2 hp + 1 of each block, those of this lane's score columns: scale of the score tile, index-free part
    f32x2 uu[NB], czz[NB];
    auto load_query = [&] {
        #pragma unroll
        for (int x = 0; x < NB; ++x) {
            const int64_t block = (int64_t)it.unit * NB + x;
            const uint32_t* fr = p.frag + block * T::FRAGS * 32 + lane;
            #pragma unroll
            for (int j = 0; j < CPL; ++j) {
                bq[x][j][0] = __ldcg(fr + 64 * j);
                bq[x][j][1] = __ldcg(fr + 64 * j + 32);
            }
            #pragma unroll
            for (int j = 0; j < T::NBZ; ++j) {
                bz[x][j][0] = __ldcg(fr + 64 * (CPL + j));
                bz[x][j][1] = __ldcg(fr + 64 * (CPL + j) + 32);
            }
            const float* hd = p.head + block * 8 + 2 * hp;
            uu[x] = f2_pack(pow2(-__float_as_int(__ldcg(hd))) * pow2(-tk), pow2(-__float_as_int(__ldcg(hd + 1))) * pow2(-tk));
            czz[x] = f2_pack(__ldcg(hd + 4), __ldcg(hd + 5));
        }
    };
    bool more = paged_next(p, cur, it);
    if (more) list_load(it, it.g0, sList);
    #pragma unroll
    for (int off = 16; off >= 1; off >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, off));
    if (lane == 0) sRed[warp] = am;
    __syncthreads();
    if (more) start_item();
    #pragma unroll
    for (int w = 0; w < W; ++w) am = fmaxf(am, sRed[w]);
    tk = pow2_to(am, 9, kTabLim);
    fill_tables();                                            // while the first codes are on their way
    __syncthreads();
    cudaGridDependencySynchronize();                          // the queries' fragments
    if (more) load_query();
    while (more) {
        // the next range's page list, while this one's codes are on their way; its item rests in shared memory
        PagedItem nx = it;
        const bool next = paged_next(p, cur, nx);
        if (next) {
            list_load(nx, nx.g0, sList + (lbuf ^ 1) * T::CHUNK);
            if (tid == 0) *sNext = nx;
        }
        // AFF: z sums onto the (x, y) sums' scale
        const float zs = pow2(max(-126, min(127, (T::EX ? 0 : 24) + tk - pow2_to(fabsf(az.dz), 0, kTabLim))));
        float M0[NB], M1[NB], l0[NB], l1[NB];
        float acc[NB][CPV + CPV / 2][4];
        #pragma unroll
        for (int x = 0; x < NB; ++x) {
            M0[x] = M1[x] = -INFINITY;
            l0[x] = l1[x] = 0.f;
            #pragma unroll
            for (int m = 0; m < CPV + CPV / 2; ++m) acc[x][m][0] = acc[x][m][1] = acc[x][m][2] = acc[x][m][3] = 0.f;
        }
        for (;;) {
            #pragma unroll 1
            while (gi < gb) {
                if (cnt) {                                    // (uniform: something was asked for)
                    ok = __all_sync(0xffffffffu, mbar_wait(&bar[stage], (phase >> stage) & 1u, kErrWaitFull)) && ok;
                    phase ^= 1u << stage;
                }
                if (cnt && ok) {
                int nv[NG];
                #pragma unroll
                for (int i = 0; i < NG; ++i) nv[i] = (cnt >> (8 * i)) & 0xff;
                // ---- scores ------------------------------------------------------------------------
                float S[NB][NG][4];
                #pragma unroll
                for (int i = 0; i < NG; ++i) {
                    float xa[NB][4], xb[NB][4], zz[NB][4];
                    uint32_t kw[2][T::KW];
                    load_k<T>(kw[0], sk + (16 * i + rho) * pitch, c);
                    load_k<T>(kw[1], sk + (16 * i + rho + 8) * pitch, c);
                    #pragma unroll
                    for (int j = 0; j < CPL; ++j) {
                        const uint2 e0 = look_xy<T>(lk, kw[0], j), e1 = look_xy<T>(lk, kw[1], j);
                        #pragma unroll
                        for (int x = 0; x < NB; ++x)
                            mma_add<T::EX>((j & 1) ? xb[x] : xa[x], e0.x, e1.x, e0.y, e1.y, bq[x][j][0], bq[x][j][1], j < 2);
                    }
                    #pragma unroll
                    for (int j = 0; j < T::NBZ; ++j) {
                        uint32_t z[4];
                        if constexpr (AFF) {
                            z[0] = k_index<T>(lk, kw[0], j, 0); z[1] = k_index<T>(lk, kw[1], j, 0);
                            z[2] = k_index<T>(lk, kw[0], j, 1); z[3] = k_index<T>(lk, kw[1], j, 1);
                        } else {
                            z[0] = look_z<T>(lk, kw[0], 2 * j); z[1] = look_z<T>(lk, kw[1], 2 * j);
                            z[2] = look_z<T>(lk, kw[0], 2 * j + 1); z[3] = look_z<T>(lk, kw[1], 2 * j + 1);
                        }
                        #pragma unroll
                        for (int x = 0; x < NB; ++x) mma_add<T::EX>(zz[x], z[0], z[1], z[2], z[3], bz[x][j][0], bz[x][j][1], j == 0);
                    }
                    #pragma unroll
                    for (int x = 0; x < NB; ++x)
                        #pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const float t = AFF ? fmaf(zz[x][y], zs, xa[x][y] + xb[x][y]) : zz[x][y] + (xa[x][y] + xb[x][y]);
                            S[x][i][y] = t + __shfl_xor_sync(0xffffffffu, t, 2);         // hi + lo columns
                        }
                }
                // ---- log2 scores, kept for the weights; running maximum; weights as B operands --------------
                uint32_t pA[NB][NG], pB[NB][NG];
                #pragma unroll
                for (int x = 0; x < NB; ++x) {
                    float mx0 = -INFINITY, mx1 = -INFINITY;
                    #pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        float (&s)[4] = S[x][i];
                        const float2 a = f2_unpack(f2_fma(f2_pack(s[0], s[1]), uu[x], czz[x]));
                        const float2 b = f2_unpack(f2_fma(f2_pack(s[2], s[3]), uu[x], czz[x]));
                        s[0] = a.x; s[1] = a.y; s[2] = b.x; s[3] = b.y;
                        if (p.raw && c < 2) {
                            float* r = p.raw + ((int64_t)it.unit * NB + x) * p.raw_us +
                                       ((int64_t)(gi << GL) + 16 * i + rho) * p.raw_h + 2 * hp;
                            #pragma unroll
                            for (int y = 0; y < 2; ++y)
                                if (2 * hp + y < p.raw_h) {
                                    if (rho < nv[i]) r[y] = s[y];
                                    if (rho + 8 < nv[i]) r[8 * p.raw_h + y] = s[2 + y];
                                }
                        }
                        if (rho >= nv[i]) s[0] = s[1] = -INFINITY;
                        if (rho + 8 >= nv[i]) s[2] = s[3] = -INFINITY;
                        mx0 = fmaxf(mx0, fmaxf(s[0], s[2]));
                        mx1 = fmaxf(mx1, fmaxf(s[1], s[3]));
                    }
                    if (__any_sync(0xffffffffu, mx0 > M0[x] || mx1 > M1[x])) {
                        #pragma unroll
                        for (int o = 4; o <= 16; o <<= 1) {
                            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
                            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
                        }
                        mx0 = fmaxf(mx0, M0[x]);
                        mx1 = fmaxf(mx1, M1[x]);
                        // (before the first token the sums are zero, or NaN from a query that is)
                        const float f0 = M0[x] == -INFINITY ? (l0[x] == 0.f ? 0.f : l0[x]) : fast_exp2(M0[x] - mx0);
                        const float f1 = M1[x] == -INFINITY ? (l1[x] == 0.f ? 0.f : l1[x]) : fast_exp2(M1[x] - mx1);
                        M0[x] = mx0;
                        M1[x] = mx1;
                        l0[x] *= f0;
                        l1[x] *= f1;
                        #pragma unroll
                        for (int m = 0; m < CPV + CPV / 2; ++m) {
                            float (&a)[4] = acc[x][m];
                            a[0] *= f0; a[1] *= f1; a[2] *= f0; a[3] *= f1;
                        }
                    }
                    // (the 2^12 is put on afterwards: score - max is exact near the maximum, + 12 would round it)
                    const float n0 = M0[x] == -INFINITY ? 0.f : M0[x], n1 = M1[x] == -INFINITY ? 0.f : M1[x];
                    #pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const float (&s)[4] = S[x][i];
                        const float p0 = fast_exp2(s[0] - n0) * 4096.f, p1 = fast_exp2(s[1] - n1) * 4096.f;
                        const float p2 = fast_exp2(s[2] - n0) * 4096.f, p3 = fast_exp2(s[3] - n1) * 4096.f;
                        l0[x] += p0 + p2;
                        l1[x] += p1 + p3;
                        const uint32_t hA = f2h2(p0, p1), hB = f2h2(p2, p3);
                        const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&hA));
                        const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&hB));
                        const uint32_t lA = f2h2(p0 - fa.x, p1 - fa.y), lB = f2h2(p2 - fb.x, p3 - fb.y);
                        pA[x][i] = movmatrix_t(c >= 2 ? lA : hA);  // column g of tokens (c, (c ^ 1) + 4)
                        pB[x][i] = movmatrix_t(c >= 2 ? lB : hB);  // column g of the same + 8
                    }
                }
                // ---- values ----------------------------------------------------------------------------
                #pragma unroll
                for (int i = 0; i < NG; ++i) {
                    uint32_t vw[4][T::VW];
                    #pragma unroll
                    for (int t = 0; t < 4; ++t) load_v<T>(vw[t], sv + (16 * i + (t & 1 ? c ^ 1 : c) + 4 * t) * pitch, g);
                    uint32_t d[NB][4];
                    #pragma unroll
                    for (int x = 0; x < NB; ++x) {
                        d[x][0] = __byte_perm(pA[x][i], 0u, 0x1010u); d[x][1] = __byte_perm(pA[x][i], 0u, 0x3232u);
                        d[x][2] = __byte_perm(pB[x][i], 0u, 0x1010u); d[x][3] = __byte_perm(pB[x][i], 0u, 0x3232u);
                    }
                    #pragma unroll
                    for (int m = 0; m < CPV; ++m) {
                        const uint2 x0 = look_xy<T>(lk, vw[0], m), x1 = look_xy<T>(lk, vw[1], m);
                        const uint2 x2 = look_xy<T>(lk, vw[2], m), x3 = look_xy<T>(lk, vw[3], m);
                        #pragma unroll
                        for (int x = 0; x < NB; ++x) {
                            mma_add<T::EX>(acc[x][m], x0.x, x0.y, x1.x, x1.y, d[x][0], d[x][1]);
                            mma_add<T::EX>(acc[x][m], x2.x, x2.y, x3.x, x3.y, d[x][2], d[x][3]);
                        }
                    }
                    #pragma unroll
                    for (int m = 0; m < CPV / 2; ++m) {
                        if constexpr (AFF) {
                            const uint32_t z0 = v_index<T>(lk, vw[0], vw[1], 2 * m), z1 = v_index<T>(lk, vw[0], vw[1], 2 * m + 1);
                            const uint32_t z2 = v_index<T>(lk, vw[2], vw[3], 2 * m), z3 = v_index<T>(lk, vw[2], vw[3], 2 * m + 1);
                            #pragma unroll
                            for (int x = 0; x < NB; ++x) {
                                float zt[4];
                                mma_zero(zt, z0, z1, z2, z3, pA[x][i], pB[x][i]);
                                #pragma unroll
                                for (int y = 0; y < 4; ++y) acc[x][CPV + m][y] += zt[y];
                            }
                        } else {
                            const uint32_t z0 = look_z<T>(lk, vw[0], 2 * m), z1 = look_z<T>(lk, vw[0], 2 * m + 1);
                            const uint32_t z2 = look_z<T>(lk, vw[1], 2 * m), z3 = look_z<T>(lk, vw[1], 2 * m + 1);
                            const uint32_t z4 = look_z<T>(lk, vw[2], 2 * m), z5 = look_z<T>(lk, vw[2], 2 * m + 1);
                            const uint32_t z6 = look_z<T>(lk, vw[3], 2 * m), z7 = look_z<T>(lk, vw[3], 2 * m + 1);
                            #pragma unroll
                            for (int x = 0; x < NB; ++x) {
                                mma_add<T::EX>(acc[x][CPV + m], z0, z1, z2, z3, d[x][0], d[x][1]);
                                mma_add<T::EX>(acc[x][CPV + m], z4, z5, z6, z7, d[x][2], d[x][3]);
                            }
                        }
                    }
                }
                }
                __syncwarp();
                cnt = cnt2;
                cnt2 = ask(gi + 2 * W, false);
                gi += W;
                stage ^= 1;
                sk = bothk - sk;
                sv = bothv - sv;
            }
            if (!ok)                                          // give what was asked for some 20 ms to arrive
                for (int x = 0; x < 4; ++x) mbar_wait(&bar[x & 1], ((phase >> (x & 1)) ^ (x >> 1)) & 1u, kErrWaitDrain, 1u << 9);
            if (gb == it.g1) break;                           // a list holds CHUNK pages; the next ones
            __syncthreads();
            list_load(it, gb, sList + lbuf * T::CHUNK);
            __syncthreads();
            start_list(gb);
        }
        // ---- hi + lo columns, the lanes, the warps ----------------------------------------------------------
        #pragma unroll
        for (int x = 0; x < NB; ++x) {
            #pragma unroll
            for (int o = 4; o <= 16; o <<= 1) {
                l0[x] += __shfl_xor_sync(0xffffffffu, l0[x], o);
                l1[x] += __shfl_xor_sync(0xffffffffu, l1[x], o);
            }
            #pragma unroll
            for (int m = 0; m < CPV + CPV / 2; ++m)
                #pragma unroll
                for (int y = 0; y < 4; ++y) acc[x][m][y] += __shfl_xor_sync(0xffffffffu, acc[x][m][y], 2);
        }
        __syncthreads();                                      // the last range's sums are read, the next one's list is there
        float* row = p.part + (int64_t)it.row * HQ * (dim + 2);
        if (next) {                                           // its first codes and its queries, before the merge
            it = *sNext;
            lbuf ^= 1;
            load_query();                                     // (first: the codes' copies fill the memory's queues)
            start_item();
        }
        more = next;
        if (c < 2) {
            #pragma unroll
            for (int x = 0; x < NB; ++x) {
                const int h0 = warp * HQ + kHQ * x + 2 * c;    // head 2c of the block; head 2c + 1 at + dim
                float* o0 = sAcc + h0 * dim;
                #pragma unroll
                for (int m = 0; m < CPV; ++m) {
                    const int t = v_triplet<T>(g, m);
                    if (t < p.m) {
                        o0[3 * t + 1] = acc[x][m][0]; o0[dim + 3 * t + 1] = acc[x][m][1];
                        o0[3 * t + 2] = acc[x][m][2]; o0[dim + 3 * t + 2] = acc[x][m][3];
                    }
                }
                #pragma unroll
                for (int m = 0; m < CPV / 2; ++m)
                    #pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int t = v_triplet<T>(g, 2 * m + y);
                        if (t < p.m) {
                            o0[3 * t] = acc[x][CPV + m][2 * y];
                            o0[dim + 3 * t] = acc[x][CPV + m][2 * y + 1];
                        }
                    }
                if (g == 0) {
                    sWm[h0] = M0[x]; sWm[h0 + 1] = M1[x];
                    sWl[h0] = l0[x]; sWl[h0 + 1] = l1[x];
                }
            }
        }
        __syncthreads();
        const float its = pow2(-tk - 12);
        for (int i = tid; i < HQ * dim; i += nthr) {
            const int h = i / dim, d = i - h * dim;
            float mx = -INFINITY, o = 0.f, ls = 0.f;
            #pragma unroll
            for (int w = 0; w < W; ++w) mx = fmaxf(mx, sWm[w * HQ + h]);
            #pragma unroll
            for (int w = 0; w < W; ++w) {
                // a warp without tokens has sum 0; a NaN sum is carried on
                const float lw = sWl[w * HQ + h], f = lw == 0.f ? 0.f : fast_exp2(sWm[w * HQ + h] - mx);
                o = fmaf(f, sAcc[(w * HQ + h) * dim + d], o);
                ls = fmaf(f, lw, ls);
            }
            // the weights carry 2^12, the tables 2^tk; AFF: sum p z = zc l + dz sum p (i - c)
            if (AFF && d % 3 == 0) o = fmaf(az.dz, o * 0x1p-12f, az.zc * (ls * 0x1p-12f));
            else o *= its;
            row[h * (dim + 2) + 2 + d] = o;
            if (d == 0) {
                row[h * (dim + 2)] = mx;
                row[h * (dim + 2) + 1] = ls * 0x1p-12f;
            }
        }
    }
}

constexpr int kJoinThreads = 384;
constexpr int kMaxGrid = 160;                  // CTAs of the attention launch, at most

// CTAs [0, blocks): one block each -- join its ranges, normalise, rotate back.  CTAs behind them (with
// weights): BATCH tokens a thread of one (sequence, KV head) each, p = exp2(score - m) / l summed over its heads.
// A unit is three round trips to memory: the ranges' (m, l), their sums, and R -- whose first rows are asked
// for before the grid dependency, thread (group kg, column d) holding rows kg, kg + groups, ... of column d.
// CTAS a multiprocessor; RB rows of R a thread asks for at a time; BATCH 0: no weights.
template <int CTAS, int RB, int BATCH>
__global__ void __launch_bounds__(kJoinThreads, CTAS) paged_join_kernel(PagedParams p, int chunks) {
    extern __shared__ float jsm[];
    const int tid = threadIdx.x, dim = p.dim, rs = dim + 2, warp = tid >> 5, lane = tid & 31;
    const int blocks = p.units * p.NB;
    if ((int)blockIdx.x < blocks) {
        float* sO = jsm;                       // [4][dim]
        float* sF = sO + kHQ * dim;            // [ranges][4] exp2(m_r - m), at most grid ranges
        float* sP = sF + kHQ * p.grid;         // [groups][4][dim] partial rotations
        __shared__ float sInv[kHQ];
        const int cols = (dim + 31) / 32 * 32, groups = kJoinThreads / cols;
        const int kg = tid / cols, d = tid - kg * cols;
        const bool mine = kg < groups && d < dim;
        float rr[RB];
        auto load_r = [&](int i0) {
            #pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int k = kg + (i0 + i) * groups;
                rr[i] = mine && k < dim ? __ldg(p.R + k * dim + d) : 0.f;
            }
        };
        load_r(0);
        int r0, r1;
        const int unit = blockIdx.x / p.NB, blk = blockIdx.x - unit * p.NB;
        unit_rows(p, unit, r0, r1);
        cudaGridDependencySynchronize();
        const float* part = p.part + ((int64_t)r0 * p.NB + blk) * kHQ * rs;
        const int64_t next = (int64_t)p.NB * kHQ * rs;         // from a range to the next
        const int nr = r1 - r0;
        if (warp < kHQ) {                       // a range without tokens has l = 0; a NaN sum is carried on
            float m[kMaxGrid / 32], l[kMaxGrid / 32], mx = -INFINITY, sum = 0.f;
            #pragma unroll
            for (int i = 0; i < kMaxGrid / 32; ++i) {
                const int r = lane + 32 * i;
                const float* q = part + r * next + warp * rs;
                m[i] = r < nr ? __ldcg(q) : 0.f;
                l[i] = r < nr ? __ldcg(q + 1) : 0.f;
            }
            #pragma unroll
            for (int i = 0; i < kMaxGrid / 32; ++i)
                if (l[i] != 0.f) mx = fmaxf(mx, m[i]);
            #pragma unroll
            for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            #pragma unroll
            for (int i = 0; i < kMaxGrid / 32; ++i) {
                const int r = lane + 32 * i;
                const float f = l[i] == 0.f ? 0.f : exp2f(m[i] - mx);
                if (r < nr) sF[r * kHQ + warp] = f;
                sum = fmaf(l[i], f, sum);
            }
            #pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (lane == 0) sInv[warp] = sum;
        }
        __syncthreads();
        for (int i = tid; i < kHQ * dim; i += kJoinThreads) {
            const int h = i / dim, x = i - h * dim;
            const float* q = part + h * rs + 2 + x;
            float o = 0.f;
            #pragma unroll 8
            for (int r = 0; r < nr; ++r) o = fmaf(sF[r * kHQ + h], __ldcg(q + r * next), o);
            sO[i] = sInv[h] == 0.f ? 0.f : o / sInv[h];
        }
        __syncthreads();
        float v[kHQ] = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 * groups < dim; i0 += RB) {
            if (i0) load_r(i0);
            #pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int k = min(kg + (i0 + i) * groups, dim - 1);         // (rr is 0 behind the last row)
                #pragma unroll
                for (int h = 0; h < kHQ; ++h) v[h] = fmaf(sO[h * dim + k], rr[i], v[h]);
            }
        }
        if (mine)
            #pragma unroll
            for (int h = 0; h < kHQ; ++h) sP[(kg * kHQ + h) * dim + d] = v[h];
        __syncthreads();
        const int b = unit / p.UH, u = unit % p.UH, hk = u / p.UG, hg = u % p.UG * p.NB + blk;
        for (int i = tid; i < kHQ * dim; i += kJoinThreads) {
            const int h = i / dim, hl = hg * kHQ + h;
            if (hl >= p.G) break;
            float o = 0.f;
            for (int x = 0; x < groups; ++x) o += sP[x * kHQ * dim + i];
            store_any(p.out, p.odt, b * p.out_bs + (int64_t)(hk * p.G + hl) * p.out_hs + (i - h * dim), o);
        }
        return;
    }
    if constexpr (BATCH > 0) {
    cudaGridDependencySynchronize();
    // ---- weights: chunks of all rows in turn (a wide table names many that are empty) ------------------
    for (int w = blockIdx.x - blocks; w < p.pg.B * p.pg.Hkv * chunks; w += gridDim.x - blocks) {
    constexpr int TOKENS = BATCH * kJoinThreads;
    const int chunk = w % chunks, bh = w / chunks, b = bh / p.pg.Hkv, hk = bh % p.pg.Hkv;
    const int L = clamp_len(p.pg, input(p.seq_lens + b));
    const int nv = p.selected ? p.n_sel << p.pg.ps_log2 : L;   // listed or dense tokens
    if (chunk * TOKENS >= nv) continue;
    // a thread's tokens: their pages, scores and weights are on their way while the heads' offsets are made
    const int end = min(nv, (chunk + 1) * TOKENS), i0 = chunk * TOKENS + tid;
    const float* raw = p.raw + ((int64_t)b * p.UH + hk * p.UG) * p.NB * p.raw_us;
    const int64_t row = ((int64_t)b * p.pg.Hkv + hk) * p.w_rs;
    int t[BATCH];
    float s[BATCH], w0[BATCH];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + u * kJoinThreads;
        t[u] = -1;
        if (i >= end) continue;
        const RangePage r = range_page(p, b, hk, i >> p.pg.ps_log2);
        const int tok = (r.logical << p.pg.ps_log2) + (i & ((1 << p.pg.ps_log2) - 1));
        if (r.page >= 0 && tok < min(L, p.w_slots)) t[u] = tok;
    }
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        s[u] = t[u] >= 0 ? __ldcg(raw + (int64_t)(i0 + u * kJoinThreads) * p.raw_h) : 0.f;
        w0[u] = t[u] >= 0 ? __ldcg(p.w_in + row + t[u]) : 0.f;
    }
    __syncthreads();                           // (the last chunk's offsets are read)
    float* sOff = jsm;                         // [G] m + log2 l
    for (int h = warp; h < p.G; h += kJoinThreads / 32) {
        int r0, r1;
        const int hb = h / kHQ;                // its block within the KV head
        unit_rows(p, b * p.UH + hk * p.UG + hb / p.NB, r0, r1);
        float mx = -INFINITY, l = 0.f;
        for (int r = r0 + lane; r < r1; r += 32) {
            const float* part = p.part + (((int64_t)r * p.NB + hb % p.NB) * kHQ + h % kHQ) * rs;
            const float mr = part[0];
            if (part[1] == 0.f) continue;
            const float nm = fmaxf(mx, mr);
            l = (l == 0.f ? 0.f : l * exp2f(mx - nm)) + part[1] * exp2f(mr - nm);
            mx = nm;
        }
        #pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, mx, off), l2 = __shfl_xor_sync(0xffffffffu, l, off);
            const float nm = fmaxf(mx, m2);
            l = (l == 0.f ? 0.f : l * exp2f(mx - nm)) + (l2 == 0.f ? 0.f : l2 * exp2f(m2 - nm));
            mx = nm;
        }
        if (lane == 0) sOff[h] = mx + log2f(l);
    }
    __syncthreads();
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        if (t[u] < 0) continue;
        float sum = exp2f(s[u] - sOff[0]);
        for (int h = 1; h < p.G; ++h)
            sum += exp2f(__ldcg(raw + h / kHQ * p.raw_us + (int64_t)(i0 + u * kJoinThreads) * p.raw_h + h % kHQ) - sOff[h]);
        p.w_out[row + t[u]] = w0[u] + sum;
    }
    }
    }
}

// ---------------------------------------------------------------------------------------------
static PagedParams paged_params(const pkv_codec* c, const pkv_paged_attn_args* a, Pages pg, int sms) {
    PagedParams p{};
    p.pg = pg;
    p.G = a->q_heads / pg.Hkv;
    // Two blocks to a unit decode each code once for eight heads, on 8 warps of 255 registers.  64 query heads over 8 KV
    // heads, one block against two: head size 96, 4 x 131072 tokens 295 -> 255 us (learned codebooks 542 -> 342); head
    // size 129, 4 x 60000 tokens 235 -> 194 us (390 -> 244).  Head sizes past 144 have no registers for it.
    p.NB = p.G > kHQ && c->dim <= 144 ? 2 : 1;
    p.UG = (p.G + p.NB * kHQ - 1) / (p.NB * kHQ);
    p.UH = pg.Hkv * p.UG;
    p.dim = c->dim;
    p.m = c->dim / 3;
    p.cb = a->pages.code_bytes;
    p.q = a->q; p.qdt = a->q_dtype; p.q_bs = a->q_batch_stride; p.q_hs = a->q_head_stride;
    p.seq_lens = a->seq_lens;
    p.selected = a->selected; p.n_sel = a->n_selected;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.out = a->out; p.odt = a->out_dtype; p.out_bs = a->out_batch_stride; p.out_hs = a->out_head_stride;
    p.w_in = a->weights; p.w_out = a->weights_out; p.w_rs = a->weights_row_stride; p.w_slots = a->weights_slots;
    p.R = c->R; p.dec_z = c->dec_z; p.dec_xy = c->dec_xy;
    p.bits_z = c->bits_z;
    p.bits_flat = c->bits_r + c->bits_theta;
    p.xy_per_z = c->xy_per_z;
    p.units = pg.B * p.UH;
    p.grid = sms < kMaxGrid ? sms : kMaxGrid;
    p.gran_log2 = p.m <= 32 ? 5 : 4;           // (launch_paged_mode)
    p.raw_h = p.G < kHQ ? p.G : kHQ;
    // room for every slot that the table (or the list) can name
    p.raw_us = ((int64_t)(a->selected ? a->n_selected : pg.max_pages) << pg.ps_log2) * p.raw_h;
    return p;
}

// Workspace: partial rows, query fragments (48 registers at most), per-head numbers, scores.
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
static size_t paged_part_bytes(const PagedParams& p) { return up256((size_t)(p.grid + p.units) * p.NB * kHQ * (p.dim + 2) * 4); }
static size_t paged_frag_bytes(const PagedParams& p) { return up256((size_t)p.units * p.NB * 48 * 32 * 4); }
static size_t paged_head_bytes(const PagedParams& p) { return up256((size_t)p.units * p.NB * 8 * 4); }

size_t paged_workspace(const pkv_codec* c, const pkv_paged_attn_args* a, Pages pg, int sms) {
    const PagedParams p = paged_params(c, a, pg, sms);
    return paged_part_bytes(p) + paged_frag_bytes(p) + paged_head_bytes(p) + (a->weights ? (size_t)p.units * p.NB * p.raw_us * 4 : 0);
}

template <class T>
static int launch_paged_as(const PagedParams& p, cudaStream_t st) {
    static_assert(T::FRAGS <= 48, "paged_frag_bytes");
    // tables from the first 64 KB boundary behind the rest (the window starts at most 1 KB into the shared space)
    const uint32_t below = 1024u + (uint32_t)pa_smem<T>(p.dim).end;
    const int smem = (int)(((below + 0xFFFFu) & ~0xFFFFu) - 1024u) + T::XY_BYTES + T::Z_BYTES + T::UPPER * T::W * T::SLOT + 128;
    static std::atomic<int> seen[64];
    int rc = allow_smem(paged_attn_kernel<T>, smem, seen);
    if (rc) return rc;
    rc = launch_behind(paged_query_kernel, (unsigned)(p.units * p.NB), kQueryThreads, (size_t)2 * kHQ * p.dim * 4, 0, st, p,
                       (int)T::AFF, T::CPL, (int)T::EX);
    if (rc) return rc;
    return launch_behind(paged_attn_kernel<T>, (unsigned)p.grid, T::THREADS, (size_t)smem, 0, st, p);
}

// EX: fp32 results -- outputs, or the running weights whatever type the outputs have -- get z from the middle bin and the
// tiles' sums added in rounded fp32 (4 x 131072 tokens: 178 us against 163; the weights' error 6e-7 relative against 2e-6
// to 6e-6). For 16-bit outputs alone the truncation of the running sums (a few 1e-6) is far below their own rounding.
// Warps by what a lane holds: 16 of 128 registers for up to 32 triplets (14 take 10 % longer, 10 take 20 %), 12 of 168
// up to 48 (16: + 9 %; 10: + 12 %), 8 of 255 up to 64 (12: + 7 %). They are what measured best, spills and all: bytes
// of spill stores with 16-bit outputs 12 to 76 (16 warps), 0 to 20 (12) and 0 (8); with EX 92 to 180, 40 to 56 and 0;
// of the two-block forms 0 to 24 and, with EX, 0 to 296.
template <int MODE, bool EX>
static int launch_paged_mode(const PagedParams& p, cudaStream_t st) {
    if (p.m <= 32)
        return p.NB == 2 ? launch_paged_as<PA<MODE, 8, 2, 8, 2, EX>>(p, st) : launch_paged_as<PA<MODE, 8, 2, 16, 1, EX>>(p, st);
    if (p.m <= 48)
        return p.NB == 2 ? launch_paged_as<PA<MODE, 12, 1, 8, 2, EX>>(p, st) : launch_paged_as<PA<MODE, 12, 1, 12, 1, EX>>(p, st);
    return launch_paged_as<PA<MODE, 16, 1, 8, 1, EX>>(p, st);
}

template <bool EX>
static int launch_paged_any(const pkv_codec* c, const PagedParams& p, cudaStream_t st) {
    const bool affine = p.bits_z <= 4 && !p.xy_per_z && (c->flags & PKV_CODEC_Z_UNIFORM);
    if (p.cb == 1) return affine ? launch_paged_mode<3, EX>(p, st) : launch_paged_mode<1, EX>(p, st);
    if (affine && p.bits_flat == 8) return launch_paged_mode<0, EX>(p, st);
    return launch_paged_mode<2, EX>(p, st);
}

template <int CTAS, int RB, int BATCH>
static int launch_join(const PagedParams& p, int64_t tokens, int sms, cudaStream_t st) {
    const int64_t per = BATCH * kJoinThreads, chunks = BATCH ? (tokens + per - 1) / per : 0, all = p.pg.B * p.pg.Hkv * chunks;
    if (all > 0x7fff0000) return PKV_ERR_UNSUPPORTED;
    const int64_t ctas = (int64_t)p.units * p.NB + (all < 16 * (int64_t)sms ? all : 16 * (int64_t)sms);
    const size_t smem = (size_t)(kHQ * p.dim + kHQ * p.grid + kJoinThreads / ((p.dim + 31) / 32 * 32) * kHQ * p.dim) * 4;
    return launch_behind(paged_join_kernel<CTAS, RB, BATCH>, (unsigned)ctas, kJoinThreads, smem, 0, st, p, (int)chunks);
}

// With weights: a third CTA per multiprocessor in place of registers where two leave more than three waves of 1536
// tokens: 128 rows of 16384 tokens 136 -> 129 us in all.  With fewer the join's rows of R count for more: 32 rows of
// 11469 to 16384 tokens (head size 129) 64.9 us with two, 68.6 with three.
static int launch_weigh(const PagedParams& p, int sms, cudaStream_t st) {
    const int64_t tokens = p.raw_us / p.raw_h;              // room for every slot that the table (or the list) can name
    const int64_t tiles = (int64_t)p.pg.B * p.pg.Hkv * ((tokens + 1535) / 1536);
    return tiles > 6 * (int64_t)sms ? launch_join<3, 8, 4>(p, tokens, sms, st) : launch_join<2, 24, 6>(p, tokens, sms, st);
}

int launch_paged_attn(const pkv_codec* c, const pkv_paged_attn_args* a, Pages pg, int sms, void* ws, cudaStream_t st) {
    PagedParams p = paged_params(c, a, pg, sms);
    uint8_t* w = static_cast<uint8_t*>(ws);
    p.part = reinterpret_cast<float*>(w);
    p.frag = reinterpret_cast<uint32_t*>(w += paged_part_bytes(p));
    p.head = reinterpret_cast<float*>(w += paged_frag_bytes(p));
    if (a->weights) p.raw = reinterpret_cast<float*>(w + paged_head_bytes(p));
    const int rc = a->out_dtype == PKV_F32 || a->weights ? launch_paged_any<true>(c, p, st) : launch_paged_any<false>(c, p, st);
    if (rc) return rc;
    return a->weights ? launch_weigh(p, sms, st) : launch_join<2, 24, 0>(p, 0, sms, st);
}

}  // namespace pkv
