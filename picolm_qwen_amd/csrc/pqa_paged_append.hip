// The new tokens of a batch into the pages: per-head RMS norm of q and k (where the layer has
// one), rotation, K and V rounded to the pages' type and written to their slots, q written
// for the attention; and the pages' key bounds.
#include <algorithm>

#include "pqa_paged_device.h"

namespace pqa {

namespace {

struct PagedAppend {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    long long ldq, ldk, ldv, ldo;
    char* kp;  // the layer's pages
    char* vp;
    const int* header;
    const PagedToken* tokens;
    const int* pages;
    const float* qn;  // [head_dim] or null
    const float* kn;
    const float* cos_tab;  // [max_pos][rot / 2] or null
    const float* sin_tab;
    int nh, n_kv, shift, style, rot;
    int vec;   // bit 0..3: rows of q, k, v, q_out are aligned to four elements
    int once;  // stores past the caches
};

// A wave takes four rows (heads) at a time, 16 lanes each, through LDS: the norm and the rotation
// pair elements that no fixed lane mapping keeps together (three pairings, any even part of the head).
// Bound by memory at prompt sizes (163 MB of fp32 prompts 35 us, 4.6 TB/s; a copy reaches 5.0) and
// by one round trip for single tokens (2.5 us). K rows are computed with the contiguous cache's arithmetic, in
// its order and without fused operations, so a page's fp16 rows have the bits that pqa_decode writes.
template <int TYPE, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppend a) {
    typedef typename PagedType<TYPE>::Io Io;
    typedef typename PagedType<TYPE>::Page Page;
    constexpr int S = HD + 4, V4 = HD / 4, N4 = (V4 + 15) / 16;
    __shared__ __attribute__((aligned(16))) float rows[16][S];
    const int lane = threadIdx.x & 63, sub = lane & 15, slot = threadIdx.x >> 4;
    float* x = rows[slot];
    const int n_tok = scalar_int(a.header, kHdTokens), heads = a.nh + 2 * a.n_kv;
    const int total = n_tok * heads;  // below 2^31 (pqa_batch_create)
    for (int u0 = blockIdx.x * 16; u0 < total; u0 += gridDim.x * 16) {
        const int u = min(u0 + slot, total - 1);  // rows past the last one: that one again, not written
        const bool live = u0 + slot < total;
        const int tok = u / heads, h = u - tok * heads;
        const int kind = h < a.nh ? 0 : h < a.nh + a.n_kv ? 1 : 2;  // q, k, v
        const int head = kind == 0 ? h : kind == 1 ? h - a.nh : h - a.nh - a.n_kv;
        const int table = a.tokens[tok].table, pos = a.tokens[tok].pos;
        const Io* src = kind == 0   ? (const Io*)a.q + (long long)tok * a.ldq
                        : kind == 1 ? (const Io*)a.k + (long long)tok * a.ldk
                                    : (const Io*)a.v + (long long)tok * a.ldv;
        float4 in[N4];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < N4; i++)
            if (sub + 16 * i < V4) in[i] = load4<Io, true>(src + head * HD + 4 * (sub + 16 * i), (a.vec >> kind) & 1);
#pragma unroll
        for (int i = 0; i < N4; i++) {
            const int f = sub + 16 * i;
            if (f < V4) {
                const float4 y = in[i];
                *(float4*)(x + 4 * f) = y;
                ss = fmaf(y.x, y.x, fmaf(y.y, y.y, fmaf(y.z, y.z, fmaf(y.w, y.w, ss))));
            }
        }
        const int page = kind == 0 ? 0 : a.pages[table + (pos >> a.shift)];
        wave_sync();
        if (kind != 2) {
            const float* nw = kind == 0 ? a.qn : a.kn;
            float sc = 1.0f;
            if (nw) {
                // k in the reference's order of summation, q (which feeds scores only) in any
                if (kind == 1) sc = rms_scale_ref_quad<HD>(x, sub & 3);
                else sc = 1.0f / sqrtf(group_sum<16>(ss) / (float)HD + 1e-6f);
                wave_sync();
#pragma unroll
                for (int i = 0; i < N4; i++) {
                    const int f = sub + 16 * i;
                    if (f < V4) {
                        const float4 y = *(const float4*)(x + 4 * f), w = *(const float4*)(nw + 4 * f);
                        *(float4*)(x + 4 * f) = float4{rms_apply(y.x, sc, w.x), rms_apply(y.y, sc, w.y),
                                                       rms_apply(y.z, sc, w.z), rms_apply(y.w, sc, w.w)};
                    }
                }
                wave_sync();
            }
            const int half = a.rot >> 1;
            const size_t at = (size_t)pos * half;
            for (int p = sub; p < half; p += 16) {
                int e0, e1;
                rope_pair(a.style, p, a.rot, e0, e1);
                float x0 = x[e0], x1 = x[e1];
                rope_rotate(x0, x1, a.cos_tab[at + p], a.sin_tab[at + p]);
                x[e0] = x0;
                x[e1] = x1;
            }
            wave_sync();
        }
        if (live) {
            if (kind == 0) {
                Io* dst = (Io*)a.q_out + (long long)tok * a.ldo + head * HD;
#pragma unroll
                for (int i = 0; i < N4; i++) {
                    const int f = sub + 16 * i;
                    if (f >= V4) continue;
                    if (a.once) store4<Io, true>(dst + 4 * f, *(const float4*)(x + 4 * f), (a.vec >> 3) & 1);
                    else store4(dst + 4 * f, *(const float4*)(x + 4 * f), (a.vec >> 3) & 1);
                }
            } else {
                const size_t row = (((unsigned)page * a.n_kv + head) << a.shift) + (pos & ((1 << a.shift) - 1));
                uint16_t* dst = (uint16_t*)(kind == 1 ? a.kp : a.vp) + row * HD;
#pragma unroll
                for (int i = 0; i < N4; i++) {
                    const int f = sub + 16 * i;
                    if (f >= V4) continue;
                    const float4 y = *(const float4*)(x + 4 * f);
                    const u32x2 v = {to_page<Page>(y.x) | (uint32_t)to_page<Page>(y.y) << 16,
                                     to_page<Page>(y.z) | (uint32_t)to_page<Page>(y.w) << 16};
                    if (a.once) __builtin_nontemporal_store(v, (u32x2*)(dst + 4 * f));
                    else *(u32x2*)(dst + 4 * f) = v;
                }
            }
        }
        wave_sync();  // the rows have been read
    }
}

// Key bounds of the pages that received rows: least and largest key of each dim over the rows in use
// (NaN left out) as whole numbers of the scale 2^(e - 6), e = floor(log2) of the largest magnitude.
// Made again from the rows, not updated, so that they hold after a page's rows were written again (a
// rejected draft) or uploaded. A workgroup per page and KV head: 16 lanes
// of 8 dims per row (HD / 8 of them used), 16 rows at a time.
template <int TYPE, int HD>
__global__ __launch_bounds__(256) void paged_bounds_kernel(const char* kp, int8_t* bounds, float* scales, const int* header,
                                                           const PagedTouched* touched, int n_kv, int shift) {
    typedef typename PagedType<TYPE>::Page Page;
    constexpr int CH = HD / 8;            // lanes per row
    constexpr int RPI = 256 / CH;         // rows at a time
    __shared__ float lo_s[RPI][HD + 1], hi_s[RPI][HD + 1];
    __shared__ float s_mx[4];
    const int tid = threadIdx.x, row = tid / CH, ch = tid - row * CH;
    const int total = scalar_int(header, kHdTouched) * n_kv;
    for (int u = blockIdx.x; u < total; u += gridDim.x) {
        const int t = u / n_kv, kvh = u - t * n_kv;
        const int page = touched[t].page, used = touched[t].used;
        const char* base = kp + (size_t)(((unsigned)page * n_kv + kvh) << shift) * (2 * HD);
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            lo[e] = __builtin_huge_valf();
            hi[e] = -__builtin_huge_valf();
        }
        if (row < RPI) {
#pragma unroll 4
            for (int r = row; r < used; r += RPI) {
                const u32x4 y = *(const u32x4*)(base + (size_t)r * (2 * HD) + 16 * ch);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float f = from_page<Page>((uint16_t)(e & 1 ? y[e >> 1] >> 16 : y[e >> 1] & 0xFFFFu));
                    lo[e] = fminf(lo[e], f);  // a NaN gives the other one
                    hi[e] = fmaxf(hi[e], f);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                lo_s[row][8 * ch + e] = lo[e];
                hi_s[row][8 * ch + e] = hi[e];
            }
        }
        __syncthreads();
        float l = __builtin_huge_valf(), h = -__builtin_huge_valf(), mx = 0.0f;
        if (tid < HD) {
            for (int r = 0; r < RPI; r++) {
                l = fminf(l, lo_s[r][tid]);
                h = fmaxf(h, hi_s[r][tid]);
            }
            mx = fmaxf(fabsf(l), fabsf(h));
        }
        mx = group_max<64>(mx);
        if ((tid & 63) == 0) s_mx[tid >> 6] = mx;
        __syncthreads();
        const int e = bound_exponent(fmaxf(fmaxf(s_mx[0], s_mx[1]), fmaxf(s_mx[2], s_mx[3])));
        const size_t at = (size_t)page * n_kv + kvh;
        if (tid < HD) {
            const float up = power2(6 - e);
            bounds[at * 2 * HD + tid] = (int8_t)fminf(fmaxf(floorf(l * up), -127.0f), 127.0f);
            bounds[at * 2 * HD + HD + tid] = (int8_t)fminf(fmaxf(ceilf(h * up), -127.0f), 127.0f);
        }
        if (tid == 0) scales[at] = power2(e - 6);
        __syncthreads();  // LDS is free again
    }
}

template <int TYPE, int HD>
hipError_t launch_append(const pqa_batch* b, int layer, const PagedAppend& a, bool captured, hipStream_t s) {
    const pqa_paged* p = b->p;
    const long long most = 8LL * p->cu_count;  // workgroups; more work takes further turns
    const long long rows = (long long)b->plan.n_tok * (p->n_heads + 2 * p->n_kv);
    const unsigned grid = (unsigned)(captured ? most : std::min(1LL << 30, (rows + 15) / 16));
    hipLaunchKernelGGL((paged_append_kernel<TYPE, HD>), dim3(grid), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p->bounds) return e;
    const long long units = (long long)b->plan.touched.size() * p->n_kv;
    const unsigned bgrid = (unsigned)(captured ? most : std::min(1LL << 30, units));
    hipLaunchKernelGGL((paged_bounds_kernel<TYPE, HD>), dim3(bgrid), dim3(256), 0, s, (const char*)a.kp,
                       p->bounds + (size_t)layer * p->layer_heads * 2 * HD, p->scales + (size_t)layer * p->layer_heads, a.header,
                       (const PagedTouched*)b->touched, p->n_kv, p->page_shift);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_type(const pqa_batch* b, int layer, const PagedAppend& a, bool captured, hipStream_t s) {
    switch (b->p->head_dim) {
#define PQA_PA(H) case H: return launch_append<TYPE, H>(b, layer, a, captured, s);
        PQA_PA(64) PQA_PA(96) PQA_PA(128) PQA_PA(160) PQA_PA(192) PQA_PA(256)
#undef PQA_PA
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_paged_append(const pqa_batch* b, int layer, const PagedRows& q, const PagedRows& k, const PagedRows& v,
                               void* q_out, long long ldo, bool captured, hipStream_t s) {
    const pqa_paged* p = b->p;
    const size_t io = (size_t)paged_io_bytes(p->type), hd = (size_t)p->head_dim;
    PagedAppend a{};
    a.q = q.p;
    a.k = k.p;
    a.v = v.p;
    a.q_out = q_out;
    a.ldq = q.ld;
    a.ldk = k.ld;
    a.ldv = v.ld;
    a.ldo = ldo;
    a.kp = p->k + (size_t)layer * p->layer_bytes;
    a.vp = p->v + (size_t)layer * p->layer_bytes;
    a.header = b->header;
    a.tokens = b->tokens;
    a.pages = b->pages;
    if (p->has_qk_norm[layer]) {
        a.qn = p->qk_norm + (size_t)layer * 2 * hd;
        a.kn = a.qn + hd;
    }
    a.cos_tab = p->rope;
    a.sin_tab = p->rope ? p->rope + (size_t)p->max_pos * (p->rot_dim / 2) : nullptr;
    a.nh = p->n_heads;
    a.n_kv = p->n_kv;
    a.shift = p->page_shift;
    a.style = p->rope_style;
    a.rot = p->rope ? p->rot_dim : 0;
    const PagedRows rows[4] = {q, k, v, {q_out, ldo}};
    for (int i = 0; i < 4; i++)
        if (((uintptr_t)rows[i].p & (4 * io - 1)) == 0 && rows[i].ld % 4 == 0) a.vec |= 1 << i;
    // Inputs are read once by anyone; what is written is soon read by the attention, unless it is more
    // than the L2s hold (32 MB): 163 MB of fp32 prompts 40.6 us through them, loads past them 38.1, stores too 36.5.
    a.once = (long long)b->plan.n_tok * (p->n_heads * (long long)io + 4LL * p->n_kv) * p->head_dim > (32LL << 20);
    switch (p->type) {
        case PQA_PAGED_F32: return launch_type<PQA_PAGED_F32>(b, layer, a, captured, s);
        case PQA_PAGED_F16: return launch_type<PQA_PAGED_F16>(b, layer, a, captured, s);
        default: return launch_type<PQA_PAGED_BF16>(b, layer, a, captured, s);
    }
}

}  // namespace pqa
