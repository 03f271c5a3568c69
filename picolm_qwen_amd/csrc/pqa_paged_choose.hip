// Which pages a query token attends to under a page budget: per KV head the `first` pages, the
// `last` ones that end with the token's own, and those of the largest scores,
//   score(page) = 2^(e_page - 6) max_h 2^(e_h - 6) sum_d max(q_hd lo_d, q_hd hi_d),
// with the page's key bounds lo, hi and the query head's row q_h as whole numbers of 7 bits and a
// sign: (nearly) the largest logit that a key of the page can have. With q split by sign the sum
// is one product of [min(q, 0), max(q, 0)] with [lo, hi] on the int8 matrix instructions, 16 pages
// by 16 heads at a time; it is a whole number below 2^22 and the scales are powers of two, so
// every score is exact and the choice is the same in any order of summation.
//
// A workgroup per token and KV head: scores to LDS as integers in the floats' order, the
// threshold by counting digits from the top, then the list in ascending order (the lower
// page where scores are equal). Bound by reading the bounds, 2 head_dim + 4 bytes per page and KV head.
#include <algorithm>

#include "pqa_paged_device.h"

namespace pqa {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));

struct PagedChoose {
    const void* q;
    long long ldq;
    const int8_t* bounds;  // the layer's
    const float* scales;
    const int* header;
    const int* token_seq;
    const PagedSeq* seqs;
    const int* pages;
    int* chosen;
    int g, n_kv, shift, select, first, last, qvec;
};

constexpr int kChooseThreads = 256, kChooseWaves = kChooseThreads / 64;

// 16 elements of a query row as whole numbers of 2^(e - 6), those of one sign (neg: the
// negative ones), the others as zero
template <class Io>
__device__ __forceinline__ intx4 signed_bytes(const Io* p, bool vec, float up, bool neg) {
    intx4 out;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float4 y = load4(p + 4 * w, vec);
        const float v[4] = {y.x, y.y, y.z, y.w};
        int word = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float r = fminf(fmaxf(rintf(v[e] * up), neg ? -127.0f : 0.0f), neg ? 0.0f : 127.0f);
            word |= ((int)r & 0xFF) << (8 * e);
        }
        out[w] = word;
    }
    return out;
}

// a float as an unsigned integer of the same order
__device__ __forceinline__ uint32_t ordered_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int TYPE, int HD>
__global__ __launch_bounds__(kChooseThreads) void paged_choose_kernel(const PagedChoose a) {
    typedef typename PagedType<TYPE>::Io Io;
    constexpr int ST = HD / 32;  // steps of 64 products
    constexpr int PB = 2;        // blocks of 16 pages at a time
    extern __shared__ uint32_t keys[];
    __shared__ int hist[256];
    __shared__ uint32_t s_lo[kChooseWaves], s_hi[kChooseWaves];
    __shared__ int s_digit, s_left, s_gt[kChooseWaves], s_eq[kChooseWaves];
    const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, g16 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cols = scalar_int(a.header, kHdTokens) * a.n_kv;
    for (int col = blockIdx.x; col < cols; col += gridDim.x) {
        const int tok = col / a.n_kv, kvh = col - tok * a.n_kv;
        const PagedSeq sq = a.seqs[scalar_int(a.token_seq, tok)];
        const int own = __builtin_amdgcn_readfirstlane((sq.len - sq.n_new + tok - sq.row0) >> a.shift);
        const int table = __builtin_amdgcn_readfirstlane(sq.table);
        const int n = own + 1;
        int* out = a.chosen + (size_t)col * a.select;
        if (n <= a.select) {  // every page
            for (int i = tid; i < a.select; i += kChooseThreads) out[i] = i < n ? i : -1;
            continue;
        }
        // scores of pages [first, n - last), in blocks of 16 PB; the heads in blocks of 16
        const int p0 = a.first, p1 = n - a.last;
        for (int i = tid; i < n; i += kChooseThreads)
            if (i < p0 || i >= p1) keys[i] = 0xFFFFFFFFu;
        uint32_t lo = 0xFFFFFFFFu, hi = 0;
        for (int h0 = 0; h0 < a.g; h0 += 16) {
            const int h = min(h0 + c16, a.g - 1);  // heads past the last one: that one again
            const Io* q = (const Io*)a.q + (long long)tok * a.ldq + (long long)(kvh * a.g + h) * HD;
            float mx = 0.0f;
#pragma unroll
            for (int st = 0; st < ST; st++) {
                const int d = 16 * ((4 * st + g16) % (HD / 16));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 y = load4(q + d + 4 * i, a.qvec);
                    mx = fmaxf(fmaxf(mx, fmaxf(fabsf(y.x), fabsf(y.y))), fmaxf(fabsf(y.z), fabsf(y.w)));
                }
            }
            const int e = bound_exponent(max_x32(max_x16(mx)));
            const float up = power2(6 - e), down = power2(e - 6);
            intx4 qb[ST];
#pragma unroll
            for (int st = 0; st < ST; st++) {
                const int chunk = 4 * st + g16, d = 16 * (chunk % (HD / 16));
                qb[st] = signed_bytes(q + d, a.qvec, up, chunk < HD / 16);
            }
            for (int b0 = p0 + 16 * PB * w; b0 < p1; b0 += 16 * PB * kChooseWaves) {
                intx4 x[PB][ST];
                int page[PB];
#pragma unroll
                for (int b = 0; b < PB; b++) page[b] = a.pages[table + min(b0 + 16 * b + c16, p1 - 1)];
#pragma unroll
                for (int b = 0; b < PB; b++) {
                    const int8_t* r = a.bounds + ((size_t)page[b] * a.n_kv + kvh) * (2 * HD) + 16 * g16;
#pragma unroll
                    for (int st = 0; st < ST; st++) x[b][st] = *(const intx4*)(r + 64 * st);
                }
                float sc[PB];
#pragma unroll
                for (int b = 0; b < PB; b++) sc[b] = a.scales[(size_t)page[b] * a.n_kv + kvh];  // of page b0 + 16 b + c16
#pragma unroll
                for (int b = 0; b < PB; b++) {
                    intx4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int st = 0; st < ST; st++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[b][st], qb[st], acc, 0, 0, 0);
                    // pages 4 g16 + j of head c16; the lane with c16 = 4 g16 + j keeps that page's
                    float mine = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float m = group_max<16>((float)acc[j] * down);
                        if (c16 == 4 * g16 + j) mine = m;
                    }
                    const int i = b0 + 16 * b + c16;
                    if ((c16 >> 2) == g16 && i < p1) {
                        const uint32_t before = h0 ? keys[i] : 0u;
                        const uint32_t key = max(before, min(ordered_bits(mine * sc[b]), 0xFFFFFFFEu));
                        keys[i] = key;
                        if (h0 + 16 >= a.g) {
                            lo = min(lo, key);
                            hi = max(hi, key);
                        }
                    }
                }
            }
        }
        // the range of the scores, so that the first digit tells them apart
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
            hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
        }
        if (lane == 0) {
            s_lo[w] = lo;
            s_hi[w] = hi;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kChooseWaves; i++) {
            lo = min(lo, s_lo[i]);
            hi = max(hi, s_hi[i]);
        }
        // the `left`-th largest of keys [p0, p1) by digits of 8 bits of key - lo, from the top:
        // key - lo has `bits` bits, of which those above `shift` are known to be `prefix`
        const int bits = hi > lo ? 32 - __clz((int)(hi - lo)) : 0;
        int left = a.select - (n - (p1 - p0));
        uint32_t prefix = 0;
        int shift = bits;
        if (left > 0)
            while (shift > 0) {
                const int width = min(8, shift), next = shift - width;
                hist[tid] = 0;
                __syncthreads();
                for (int i = p0 + tid; i < p1; i += kChooseThreads) {
                    const uint32_t k = keys[i] - lo;
                    if (shift >= 32 || (k >> shift) == prefix) atomicAdd(&hist[(k >> next) & ((1u << width) - 1)], 1);
                }
                __syncthreads();
                if (w == 0) {  // lane l: digits 4 l .. 4 l + 3; the sum of all larger ones by a scan
                    int c[4], sum = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) sum += c[j] = hist[4 * lane + j];
                    int above = sum;  // of this lane's digits and all higher lanes'
#pragma unroll
                    for (int d = 1; d < 64; d <<= 1) {
                        const int y = __shfl_down(above, d);
                        if (lane + d < 64) above += y;
                    }
                    int over = above - sum;  // strictly above this lane's digits
#pragma unroll
                    for (int j = 3; j >= 0; j--) {
                        if (over < left && left <= over + c[j]) {
                            s_digit = 4 * lane + j;
                            s_left = left - over;
                        }
                        over += c[j];
                    }
                }
                __syncthreads();
                prefix = prefix << width | (uint32_t)s_digit;
                left = s_left;
                shift = next;
            }
        // keys above lo + prefix are chosen, and the first `left` that equal it; each wave lists a
        // run of the pages behind what the waves before it found
        const uint32_t at = left > 0 ? lo + prefix : 0xFFFFFFFFu;  // left == 0: the forced pages alone
        const bool none = left <= 0;
        const int run = (n + kChooseWaves * 64 - 1) / (kChooseWaves * 64) * 64, r0 = w * run, r1 = min(n, r0 + run);
        int gt = 0, eq = 0;
        for (int i = r0 + lane; i < r1; i += 64) {
            const uint32_t k = keys[i];
            gt += none ? k == 0xFFFFFFFFu : k > at;
            eq += !none && k == at;
        }
        for (int d = 32; d; d >>= 1) {
            gt += __shfl_xor(gt, d);
            eq += __shfl_xor(eq, d);
        }
        if (lane == 0) {
            s_gt[w] = gt;
            s_eq[w] = eq;
        }
        __syncthreads();
        int put = 0, same = 0;  // listed, and equal ones met, before this wave's run
        for (int i = 0; i < w; i++) {
            put += s_gt[i] + min(s_eq[i], max(0, left - same));
            same += s_eq[i];
        }
        const unsigned long long below = (1ull << lane) - 1;
        for (int i0 = r0; i0 < r1; i0 += 64) {
            const int i = i0 + lane;
            const uint32_t k = i < r1 ? keys[i] : 0u;
            const bool is = i < r1 && !none && k == at;
            const unsigned long long equal = __ballot(is);
            const bool take = i < r1 && ((none ? k == 0xFFFFFFFFu : k > at) || (is && same + __popcll(equal & below) < left));
            const unsigned long long taken = __ballot(take);
            const int to = put + __popcll(taken & below);
            if (take && to < a.select) out[to] = i;
            put += __popcll(taken);
            same += __popcll(equal);
        }
        __syncthreads();  // LDS is free again
    }
}

template <int TYPE, int HD>
hipError_t launch_choose(const PagedChoose& a, unsigned grid, size_t lds, hipStream_t s) {
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)paged_choose_kernel<TYPE, HD>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 kPagedMaxChoice * 4);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((paged_choose_kernel<TYPE, HD>), dim3(grid), dim3(kChooseThreads), lds, s, a);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_type(int hd, const PagedChoose& a, unsigned grid, size_t lds, hipStream_t s) {
    switch (hd) {
#define PQA_PC(H) case H: return launch_choose<TYPE, H>(a, grid, lds, s);
        PQA_PC(64) PQA_PC(96) PQA_PC(128) PQA_PC(160) PQA_PC(192) PQA_PC(256)
#undef PQA_PC
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_paged_choose(const pqa_batch* b, int layer, const PagedRows& q, int select, int first, int last, int* chosen,
                               bool captured, hipStream_t s) {
    const pqa_paged* p = b->p;
    const size_t io = (size_t)paged_io_bytes(p->type);
    PagedChoose a{};
    a.q = q.p;
    a.ldq = q.ld;
    a.bounds = p->bounds + (size_t)layer * p->layer_heads * 2 * p->head_dim;
    a.scales = p->scales + (size_t)layer * p->layer_heads;
    a.header = b->header;
    a.token_seq = b->token_seq;
    a.seqs = b->seqs;
    a.pages = b->pages;
    a.chosen = chosen;
    a.g = p->group;
    a.n_kv = p->n_kv;
    a.shift = p->page_shift;
    a.select = select;
    a.first = first;
    a.last = last;
    a.qvec = ((uintptr_t)q.p & (4 * io - 1)) == 0 && q.ld % 4 == 0;
    int longest = 0;
    if (captured) longest = b->shape.max_seq_pages;
    else
        for (const PagedSeq& sq : b->plan.seqs)
            if (sq.n_new) longest = std::max(longest, (sq.len + p->page_size - 1) / p->page_size);
    if (longest > kPagedMaxChoice) return hipErrorInvalidValue;
    const size_t lds = (size_t)longest * 4;
    const long long most = 16LL * p->cu_count;
    const unsigned grid = (unsigned)(captured ? most : std::min<long long>(most, (long long)b->plan.n_tok * p->n_kv));
    switch (p->type) {
        case PQA_PAGED_F32: return launch_type<PQA_PAGED_F32>(p->head_dim, a, grid, lds, s);
        case PQA_PAGED_F16: return launch_type<PQA_PAGED_F16>(p->head_dim, a, grid, lds, s);
        default: return launch_type<PQA_PAGED_BF16>(p->head_dim, a, grid, lds, s);
    }
}

}  // namespace pqa
