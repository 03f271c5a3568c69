// Kernels that choose the pages of a batch's tokens under a page budget (pqa_paged_choose.h).
#include <algorithm>

#include "pqa_paged_choose.h"

namespace pqa {

namespace {

template <int TYPE, int HD>
__global__ __launch_bounds__(choose_threads<HD>()) void paged_choose_kernel(const PagedChoose a) {
    extern __shared__ uint32_t lds_keys[];
    __shared__ ListScratch scratch;
    __shared__ int s_flag;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), threads = blockDim.x, waves = threads >> 6;
    // the tokens whose number is a multiple of the group come first, in one run: most of the others
    // leave at once, and would leave CUs idle in between
    const int n_tok = scalar_int(a.header, kHdTokens), heads = (n_tok + a.group - 1) / a.group;
    for (int u = blockIdx.x; u < heads * a.group * a.n_kv * a.parts; u += gridDim.x) {
        // a column's parts lie next to each other, so on different dies
        const int col = u / a.parts, part = u - col * a.parts;
        const int kvh = col % a.n_kv, v = col / a.n_kv, tok = v % heads * a.group + v / heads;
        if (tok >= n_tok) continue;
        const int* token = a.tokens + 4 * (size_t)tok;
        const int table = scalar_int(token, 0), pos = scalar_int(token, 1);
        if (scalar_int(token, 2) % a.group) continue;  // another token's workgroup has it
        const int nt = min(a.group, scalar_int(token, 3));
        const int top = ((pos + nt - 1) >> a.shift) + 1;  // pages that the last of the tokens sees
        if (top > a.select) {
            const int all0 = a.first, all1 = top - a.last;
            const int p0 = all0 + (int)((long long)(all1 - all0) * part / a.parts);
            const int p1 = all0 + (int)((long long)(all1 - all0) * (part + 1) / a.parts);
            score_pages<TYPE, HD, (HD <= 128 ? 4 : 2)>(a, lds_keys, tok, nt, kvh, table, p0, p1, w, waves);
            __syncthreads();
            if (a.parts > 1) {
                uint32_t* to = a.part_keys + (size_t)col * a.stride;
                for (int i = p0 + tid; i < p1; i += threads)
                    __hip_atomic_store(to + i, lds_keys[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const bool last = last_of(a.counters + col, a.parts, &s_flag);
                if (last)
                    for (int i = all0 + tid; i < all1; i += threads)
                        lds_keys[i] = __hip_atomic_load(to + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
                if (!last) continue;
            }
        } else if (part) {
            continue;
        }
        // a list per token: short ones a wave each
        for (int t = 0; t < nt; t++) {
            const int n = ((pos + t) >> a.shift) + 1;
            if (n > a.select && n > kWaveKeys) continue;
            if (t % waves != w) continue;
            int* out = a.chosen + ((size_t)(tok + t) * a.n_kv + kvh) * a.select;
            if (n <= a.select) {  // every page
                for (int i = lane; i < a.select; i += 64) out[i] = i < n ? i : -1;
            } else {
                const Keys keys = {lds_keys + t * a.stride, a.first, n - a.last, n};
                if (n <= 256) choose_by_wave<4>(keys, a.select, lane, out);
                else if (n <= 512) choose_by_wave<8>(keys, a.select, lane, out);
                else if (n <= 768) choose_by_wave<12>(keys, a.select, lane, out);
                else choose_by_wave<16>(keys, a.select, lane, out);
            }
        }
        for (int t = 0; t < nt; t++) {
            const int n = ((pos + t) >> a.shift) + 1;
            if (n <= a.select || n <= kWaveKeys) continue;
            int* out = a.chosen + ((size_t)(tok + t) * a.n_kv + kvh) * a.select;
            const Keys keys = {lds_keys + t * a.stride, a.first, n - a.last, n};
            choose_by_block(keys, a.select, scratch, w, waves, out);
        }
        __syncthreads();  // LDS is free again
    }
}

template <int TYPE, int HD>
hipError_t launch_choose(const PagedChoose& a, unsigned grid, size_t lds, hipStream_t s) {
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)paged_choose_kernel<TYPE, HD>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (kPagedMaxChoice + 1) * 4);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((paged_choose_kernel<TYPE, HD>), dim3(grid), dim3(a.group > 1 ? 512 : choose_threads<HD>()), lds, s, a);
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

PagedChoose choose_arguments(const pqa_batch* b, int layer, const PagedRows& q, int select, int first, int last, int* chosen,
                             bool captured) {
    const pqa_paged* p = b->p;
    const size_t io = (size_t)paged_io_bytes(p->type);
    PagedChoose a{};
    a.q = q.p;
    a.ldq = q.ld;
    a.bounds = p->bounds + (size_t)layer * p->layer_heads * 2 * p->head_dim;
    a.scales = p->scales + (size_t)layer * p->layer_heads;
    a.header = b->header;
    a.tokens = (const int*)b->tokens;
    a.pages = b->pages;
    a.chosen = chosen;
    a.g = p->group;
    a.n_kv = p->n_kv;
    a.shift = p->page_shift;
    a.select = select;
    a.first = first;
    a.last = last;
    a.qvec = ((uintptr_t)q.p & (4 * io - 1)) == 0 && q.ld % 4 == 0;
    int longest = 0, seqs = 0;
    if (captured) longest = b->shape.max_seq_pages;
    else
        for (const PagedSeq& sq : b->plan.seqs)
            if (sq.n_new) {
                longest = std::max(longest, (sq.len + p->page_size - 1) / p->page_size);
                seqs++;
            }
    a.single = !captured && b->plan.n_tok == seqs;
    a.stride = longest | 1;  // odd: the tokens' keys of one page lie in different banks
    a.group = a.single ? 1 : std::max(1, std::min(a.g > 16 ? 1 : 16 / a.g, kChooseBytes / (4 * a.stride)));
    // Few columns share out many pages: one CU's loads take longer than passing the keys on does, some 3 us
    // (choice and attention of one token, bf16, 32 / 8 heads of 128, 32 pages of 16 chosen: behind 131072
    // positions 132 us unshared, 37 shared; 20000 34 and 30; 9000, not shared, 24).
    const long long columns = (long long)(captured ? b->shape.max_tokens : b->plan.n_tok) * p->n_kv;
    a.parts = 1;
    if (columns && (a.single || captured))
        a.parts = (int)std::max<long long>(1, std::min<long long>(p->cu_count / columns, longest / kPartPages));
    if (a.parts > 1 && columns * a.stride > (long long)paged_narrow_slots(b->shape) * 16 * (p->head_dim + 2)) a.parts = 1;
    if (a.parts > 1) a.group = 1;
    a.part_keys = (uint32_t*)b->part_narrow;
    a.counters = b->counters;
    return a;
}

hipError_t launch_paged_choose(const pqa_batch* b, const PagedChoose& a, bool captured, hipStream_t s) {
    const pqa_paged* p = b->p;
    const size_t lds = (size_t)a.group * a.stride * 4;
    const long long most = 16LL * p->cu_count;
    const long long units = ((long long)b->plan.n_tok + a.group) * p->n_kv * a.parts;
    const unsigned grid = (unsigned)(captured ? most : std::min<long long>(1 << 30, units));
    switch (p->type) {
        case PQA_PAGED_F32: return launch_type<PQA_PAGED_F32>(p->head_dim, a, grid, lds, s);
        case PQA_PAGED_F16: return launch_type<PQA_PAGED_F16>(p->head_dim, a, grid, lds, s);
        default: return launch_type<PQA_PAGED_BF16>(p->head_dim, a, grid, lds, s);
    }
}

}  // namespace pqa
