// pkv_paged_attn.cu -- decode attention of one token per sequence over a paged code cache.
//
//   out[b, h] = R^T ( sum_t p_t V^(t) / sum_t p_t ),   p_t = exp(scale (R q) . K^(t) - max)
//
// over the sequence's tokens or those of listed pages; optionally weights_out[t] = weights[t] +
// sum_h p_t / sum p.  Two launches: paged_attn_kernel leaves one partial state per (CTA, unit) range,
// paged_join_kernel joins a unit's ranges, normalises and rotates back (and, in further CTAs, adds the
// weights from the scores that the first launch kept).

#include "pkv_paged.cuh"

namespace pkv {

constexpr int kHQ = 4;                         // query heads per unit

// One warp per granule, lanes over triplets, fp32 throughout.
__global__ void __launch_bounds__(256) paged_attn_kernel(PagedParams p) {
    extern __shared__ float psm[];
    const int dim = p.dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
    float* sQ = psm;                           // [4][dim] scaled rotated queries
    float* sAcc = sQ + kHQ * dim;              // [warps][4][dim]
    float* sM = sAcc + nw * kHQ * dim;         // [warps][4], then l
    float* sL = sM + nw * kHQ;
    PagedCursor cur = paged_begin(p);
    PagedItem it;
    while (paged_next(p, cur, it)) {
        __syncthreads();
        const int L = clamp_len(p.pg, p.seq_lens[it.b]);
        for (int i = warp; i < kHQ * dim; i += nw) {
            const int h = i / dim, k = i % dim, hl = it.hg * kHQ + h;
            float a = 0.f;
            if (hl < p.G)
                for (int d = lane; d < dim; d += 32)
                    a = fmaf(__ldg(p.R + k * dim + d),
                             load_any(p.q, p.qdt, it.b * p.q_bs + (int64_t)(it.hk * p.G + hl) * p.q_hs + d), a);
            #pragma unroll
            for (int off = 16; off >= 1; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
            if (lane == 0) sQ[i] = a * p.scale_log2;
        }
        __syncthreads();
        float M[kHQ], l[kHQ], acc[kHQ][6];
        #pragma unroll
        for (int h = 0; h < kHQ; ++h) {
            M[h] = -INFINITY;
            l[h] = 0.f;
            #pragma unroll
            for (int i = 0; i < 6; ++i) acc[h][i] = 0.f;
        }
        for (int gi = it.g0 + warp; gi < it.g1; gi += nw) {
            const Granule g = granule_at(p, it.b, it.hk, gi);
            if (g.page < 0) continue;
            for (int r = 0; r < kGranule && g.tok + r < L; ++r) {
                const int64_t off = slot_offset(p.pg, g.page, it.hk, g.slot + r);
                float s[kHQ] = {0.f, 0.f, 0.f, 0.f}, vz[2], vx[2], vy[2];
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = lane + 32 * i;
                    vz[i] = vx[i] = vy[i] = 0.f;
                    if (j >= p.m) continue;
                    uint32_t kc, vc;
                    if (p.cb == 1) {
                        kc = p.pg.k[off + j];
                        vc = p.pg.v[off + j];
                    } else {
                        kc = reinterpret_cast<const uint16_t*>(p.pg.k + off)[j];
                        vc = reinterpret_cast<const uint16_t*>(p.pg.v + off)[j];
                    }
                    const uint32_t cm = (1u << (p.bits_z + p.bits_flat)) - 1u, fm = (1u << p.bits_flat) - 1u;
                    kc &= cm;
                    vc &= cm;
                    const float kz = p.dec_z[kc >> p.bits_flat];
                    const float2 kxy = reinterpret_cast<const float2*>(p.dec_xy)[p.xy_per_z ? kc : kc & fm];
                    const float2 vxy = reinterpret_cast<const float2*>(p.dec_xy)[p.xy_per_z ? vc : vc & fm];
                    vz[i] = p.dec_z[vc >> p.bits_flat];
                    vx[i] = vxy.x;
                    vy[i] = vxy.y;
                    #pragma unroll
                    for (int h = 0; h < kHQ; ++h) {
                        const float* qv = sQ + h * dim + 3 * j;
                        s[h] = fmaf(qv[0], kz, fmaf(qv[1], kxy.x, fmaf(qv[2], kxy.y, s[h])));
                    }
                }
                #pragma unroll
                for (int h = 0; h < kHQ; ++h)
                    #pragma unroll
                    for (int o = 16; o >= 1; o >>= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], o);
                if (p.raw && lane == 0)
                    for (int h = 0; h < p.raw_h; ++h)
                        p.raw[(int64_t)it.unit * p.raw_us + ((int64_t)gi * kGranule + r) * p.raw_h + h] = s[h];
                #pragma unroll
                for (int h = 0; h < kHQ; ++h) {
                    const float n = fmaxf(M[h], s[h]), f = exp2f(M[h] - n), e = exp2f(s[h] - n);
                    M[h] = n;
                    l[h] = fmaf(l[h], f, e);
                    #pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        acc[h][3 * i] = fmaf(acc[h][3 * i], f, e * vz[i]);
                        acc[h][3 * i + 1] = fmaf(acc[h][3 * i + 1], f, e * vx[i]);
                        acc[h][3 * i + 2] = fmaf(acc[h][3 * i + 2], f, e * vy[i]);
                    }
                }
            }
        }
        for (int h = 0; h < kHQ; ++h) {
            for (int i = 0; i < 6; ++i) {
                const int d = 3 * (lane + 32 * (i / 3)) + i % 3;
                if (d < dim) sAcc[(warp * kHQ + h) * dim + d] = acc[h][i];
            }
            if (lane == 0) {
                sM[warp * kHQ + h] = M[h];
                sL[warp * kHQ + h] = l[h];
            }
        }
        __syncthreads();
        float* row = p.part + (int64_t)it.row * kHQ * (dim + 2);
        for (int i = tid; i < kHQ * dim; i += blockDim.x) {
            const int h = i / dim, d = i % dim;
            float mx = -INFINITY, o = 0.f, ls = 0.f;
            for (int w = 0; w < nw; ++w) mx = fmaxf(mx, sM[w * kHQ + h]);
            for (int w = 0; w < nw; ++w) {
                const float f = sL[w * kHQ + h] == 0.f ? 0.f : exp2f(sM[w * kHQ + h] - mx);   // (NaN sums stay)
                o = fmaf(f, sAcc[(w * kHQ + h) * dim + d], o);
                ls = fmaf(f, sL[w * kHQ + h], ls);
            }
            row[h * (dim + 2) + 2 + d] = o;
            if (d == 0) {
                row[h * (dim + 2)] = mx;
                row[h * (dim + 2) + 1] = ls;
            }
        }
    }
}

// The ranges of a unit: partial rows [r0, r1), empty for a unit without granules.  Whole warps.
__device__ inline void unit_rows(const PagedParams& p, int unit, int& r0, int& r1, int& n) {
    const int b = unit / p.UH;
    int64_t before, total;
    granule_line(p, b, before, total);
    n = granules_of(p, b);
    r0 = r1 = 0;
    if (n == 0) return;
    const int64_t gd = min((int64_t)p.grid, total);
    const int64_t a = before + (int64_t)(unit % p.UH) * n;
    r0 = (int)(((a + 1) * gd - 1) / total) + unit;
    r1 = (int)(((a + n) * gd - 1) / total) + unit + 1;
}

constexpr int kJoinThreads = 256;
constexpr int kWeighTokens = 2048;             // tokens per CTA of the weight pass

// CTAs [0, units): one unit each -- join its ranges, normalise, rotate back.  CTAs behind them (with
// weights): kWeighTokens tokens of one (sequence, KV head) each, p = exp2(score - m) / l summed over its heads.
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(PagedParams p, int chunks) {
    extern __shared__ float jsm[];
    const int tid = threadIdx.x, dim = p.dim, rs = dim + 2;
    cudaGridDependencySynchronize();
    if ((int)blockIdx.x < p.units) {
        float* sO = jsm;                       // [4][dim]
        int r0, r1, n;
        const int unit = blockIdx.x;
        unit_rows(p, unit, r0, r1, n);
        for (int i = tid; i < kHQ * dim; i += kJoinThreads) {
            const int h = i / dim, d = i % dim;
            const float* part = p.part + ((int64_t)r0 * kHQ + h) * rs;
            float mx = -INFINITY, l = 0.f, o = 0.f;
            for (int r = r0; r < r1; ++r, part += kHQ * rs) {
                const float mr = part[0];
                if (part[1] == 0.f) continue;       // no token (a NaN sum is carried on)
                const float nm = fmaxf(mx, mr), f0 = l == 0.f ? 0.f : exp2f(mx - nm), f1 = exp2f(mr - nm);
                mx = nm;
                l = fmaf(l, f0, part[1] * f1);
                o = fmaf(o, f0, part[2 + d] * f1);
            }
            sO[i] = l == 0.f ? 0.f : o / l;
        }
        __syncthreads();
        const int b = unit / p.UH, u = unit % p.UH, hk = u / p.UG, hg = u % p.UG;
        for (int i = tid; i < kHQ * dim; i += kJoinThreads) {
            const int h = i / dim, d = i % dim, hl = hg * kHQ + h;
            if (hl >= p.G) break;
            float v = 0.f;
            for (int k = 0; k < dim; ++k) v = fmaf(sO[h * dim + k], __ldg(p.R + k * dim + d), v);
            store_any(p.out, p.odt, b * p.out_bs + (int64_t)(hk * p.G + hl) * p.out_hs + d, v);
        }
        return;
    }
    // ---- weights -----------------------------------------------------------------------------
    const int w = blockIdx.x - p.units, chunk = w % chunks, bh = w / chunks, b = bh / p.pg.Hkv, hk = bh % p.pg.Hkv;
    const int L = clamp_len(p.pg, p.seq_lens[b]);
    const int nv = granules_of(p, b) * kGranule;   // listed or dense tokens
    if (chunk * kWeighTokens >= nv) return;
    float* sOff = jsm;                         // [G] m + log2 l
    const int warp = tid >> 5, lane = tid & 31;
    for (int h = warp; h < p.G; h += kJoinThreads / 32) {
        int r0, r1, n;
        unit_rows(p, b * p.UH + hk * p.UG + h / kHQ, r0, r1, n);
        float mx = -INFINITY, l = 0.f;
        for (int r = r0 + lane; r < r1; r += 32) {
            const float* part = p.part + ((int64_t)r * kHQ + h % kHQ) * rs;
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
    const int end = min(nv, (chunk + 1) * kWeighTokens);
    for (int i = chunk * kWeighTokens + tid; i < end; i += kJoinThreads) {
        int t = i;
        if (p.selected) {
            const Granule g = granule_at(p, b, hk, i >> 4);
            if (g.page < 0) continue;
            t = g.tok + (i & 15);
        } else if (t < L && page_of(p.pg, b, t >> p.pg.ps_log2) < 0) {
            continue;
        }
        if (t >= L || t >= p.w_slots) continue;
        float sum = 0.f;
        for (int h = 0; h < p.G; ++h) {
            const int64_t u = (int64_t)b * p.UH + hk * p.UG + h / kHQ;
            sum += exp2f(p.raw[u * p.raw_us + (int64_t)i * p.raw_h + h % kHQ] - sOff[h]);
        }
        const int64_t at = ((int64_t)b * p.pg.Hkv + hk) * p.w_rs + t;
        p.w_out[at] = p.w_in[at] + sum;
    }
}

// ---------------------------------------------------------------------------------------------
static PagedParams paged_params(const pkv_codec* c, const pkv_paged_attn_args* a, Pages pg, int sms) {
    PagedParams p{};
    p.pg = pg;
    p.Hq = a->q_heads;
    p.G = a->q_heads / pg.Hkv;
    p.HQ = kHQ;
    p.UG = (p.G + kHQ - 1) / kHQ;
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
    p.grid = sms;
    p.raw_h = p.G < kHQ ? p.G : kHQ;
    // room for every slot that the table (or the list) can name
    p.raw_us = ((int64_t)(a->selected ? a->n_selected : pg.max_pages) << pg.ps_log2) * p.raw_h;
    return p;
}

static size_t paged_part_bytes(const PagedParams& p) {
    return ((size_t)(p.grid + p.units) * kHQ * (p.dim + 2) * 4 + 255) / 256 * 256;
}

size_t paged_workspace(const pkv_codec* c, const pkv_paged_attn_args* a, Pages pg, int sms) {
    const PagedParams p = paged_params(c, a, pg, sms);
    return paged_part_bytes(p) + (a->weights ? (size_t)p.units * p.raw_us * 4 : 0);
}

int launch_paged_attn(const pkv_codec* c, const pkv_paged_attn_args* a, Pages pg, int sms, void* ws, cudaStream_t st) {
    PagedParams p = paged_params(c, a, pg, sms);
    p.part = static_cast<float*>(ws);
    if (a->weights) p.raw = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + paged_part_bytes(p));
    constexpr int threads = 256;
    const size_t smem = (size_t)(kHQ * p.dim + threads / 32 * kHQ * (p.dim + 2)) * 4;
    paged_attn_kernel<<<p.grid, threads, smem, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return PKV_ERR_CUDA;
    const int chunks = a->weights ? (int)((p.raw_us / p.raw_h + kWeighTokens - 1) / kWeighTokens) : 0;
    const int64_t ctas = p.units + (int64_t)pg.B * pg.Hkv * chunks;
    if (ctas > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = (size_t)(kHQ * p.dim > 16 ? kHQ * p.dim : 16) * 4;   // outputs, or one value per head
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel, p, chunks) == cudaSuccess ? PKV_OK : PKV_ERR_CUDA;
}

}  // namespace pkv
