// The paged cache's C entry points (include/pqa.h): argument checks, ownership, the batch's
// upload. Kernels: pqa_paged_append.hip, pqa_paged_attn.hip, pqa_paged_choose.hip.
#include "pqa_paged.h"

#include <algorithm>
#include <cstring>
#include <new>

#include "pqa_internal.h"

using pqa::PagedFault;
using pqa::set_err;

namespace {

int fail(pqa_paged* p, int code, const std::string& msg) {
    if (!p) return set_err(nullptr, code, msg);
    p->err = msg;
    return code;
}

int hip_fail(pqa_paged* p, hipError_t e, const std::string& what) {
    return fail(p, e == hipErrorOutOfMemory ? PQA_ERR_NOMEM : PQA_ERR_HIP, what + ": " + hipGetErrorString(e));
}

// The handle's device for the length of a call, whatever the caller's thread has selected.
struct OnDevice {
    int before = -1;
    hipError_t err = hipSuccess;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// Nothing throws across the ABI: the only exceptions here are allocations on the host.
template <class F>
int guarded(pqa_paged* p, const char* fn, F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        try {
            return fail(p, PQA_ERR_NOMEM, std::string(fn) + ": out of host memory");
        } catch (...) {
            return PQA_ERR_NOMEM;
        }
    } catch (...) {
        return PQA_ERR_NOMEM;
    }
}

template <typename T>
hipError_t dev_alloc(T** p, size_t bytes) {
    return hipMalloc((void**)p, std::max<size_t>(bytes, 16));
}

void free_paged(pqa_paged* p) {
    if (!p) return;
    OnDevice on(p->device);
    (void)hipDeviceSynchronize();
    if (p->owned) {
        void* bufs[] = {p->k, p->v, p->bounds, p->scales};
        for (void* b : bufs)
            if (b) (void)hipFree(b);
    }
    if (p->rope) (void)hipFree(p->rope);
    if (p->qk_norm) (void)hipFree(p->qk_norm);
    delete p;
}

void free_batch(pqa_batch* b) {
    if (!b) return;
    OnDevice on(b->device);
    (void)hipDeviceSynchronize();
    if (b->mem) (void)hipFree(b->mem);
    for (int i = 0; i < 2; i++) {
        if (b->stage[i]) (void)hipHostFree(b->stage[i]);
        if (b->copied[i]) (void)hipEventDestroy(b->copied[i]);
    }
    delete b;
}

hipError_t is_captured(hipStream_t s, bool* captured) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    const hipError_t e = hipStreamIsCapturing(s, &st);
    *captured = st != hipStreamCaptureStatusNone;
    return e;
}

}  // namespace

extern "C" int pqa_paged_create(pqa_paged** out, int n_layers, int n_pages, int page_size, int n_heads, int n_kv_heads,
                                int head_dim, int type, int with_bounds, void* key_pages, void* val_pages, int8_t* key_bounds,
                                float* key_scales) {
    static const char* fn = "pqa_paged_create";
    return guarded(nullptr, fn, [&]() -> int {
        const std::string name = fn;
        if (!out) return fail(nullptr, PQA_ERR_ARG, name + ": out is NULL");
        *out = nullptr;
        if (n_layers <= 0 || n_pages <= 0 || n_heads <= 0 || n_kv_heads <= 0)
            return fail(nullptr, PQA_ERR_ARG, name + ": sizes must be positive");
        if (n_heads % n_kv_heads != 0) return fail(nullptr, PQA_ERR_ARG, name + ": n_heads must be a multiple of n_kv_heads");
        if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
            return fail(nullptr, PQA_ERR_UNSUPPORTED, name + ": page_size must be 16, 32, 64, 128 or 256");
        if (!pqa::paged_head_dim(head_dim))
            return fail(nullptr, PQA_ERR_UNSUPPORTED, name + ": head_dim must be 64, 96, 128, 160, 192 or 256");
        if (type < PQA_PAGED_F32 || type > PQA_PAGED_BF16) return fail(nullptr, PQA_ERR_ARG, name + ": bad type");
        // a layer's rows are counted in 31 bits (their bytes in 64); heads * dims in 31 too
        if ((long long)n_pages * n_kv_heads * page_size >= (1LL << 31) || (long long)n_heads * head_dim >= (1LL << 24))
            return fail(nullptr, PQA_ERR_UNSUPPORTED, name + ": more than 2^31 rows per layer or 2^24 elements per token");
        const bool given = key_pages || val_pages || key_bounds || key_scales;
        if (given && (!key_pages || !val_pages || (with_bounds && (!key_bounds || !key_scales)) ||
                      (!with_bounds && (key_bounds || key_scales))))
            return fail(nullptr, PQA_ERR_ARG, name + ": give all of the cache's memory or none of it");
        if (((uintptr_t)key_pages | (uintptr_t)val_pages | (uintptr_t)key_bounds) & 15u || (uintptr_t)key_scales & 3u)
            return fail(nullptr, PQA_ERR_ARG, name + ": misaligned memory (pages and bounds 16 bytes, scales 4)");
        pqa_paged* p = new pqa_paged();
        p->n_layers = n_layers;
        p->n_pages = n_pages;
        p->page_size = page_size;
        while ((1 << p->page_shift) < page_size) p->page_shift++;
        p->n_heads = n_heads;
        p->n_kv = n_kv_heads;
        p->group = n_heads / n_kv_heads;
        p->head_dim = head_dim;
        p->type = type;
        p->layer_heads = (size_t)n_pages * n_kv_heads;
        p->layer_bytes = p->layer_heads * page_size * head_dim * 2;
        p->owned = !given;
        p->k = (char*)key_pages;
        p->v = (char*)val_pages;
        p->bounds = key_bounds;
        p->scales = key_scales;
        hipError_t e = hipGetDevice(&p->device);
        int cus = 0;
        if (e == hipSuccess && hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, p->device) == hipSuccess && cus > 0)
            p->cu_count = cus;
        try {
            p->has_qk_norm.assign(n_layers, 0);
        } catch (...) {
            delete p;
            throw;
        }
        const size_t all = (size_t)n_layers * p->layer_bytes, heads = (size_t)n_layers * p->layer_heads;
        if (e == hipSuccess && p->owned) {
            e = dev_alloc(&p->k, all);
            if (e == hipSuccess) e = dev_alloc(&p->v, all);
            if (e == hipSuccess) e = hipMemset(p->k, 0, all);
            if (e == hipSuccess) e = hipMemset(p->v, 0, all);
            if (with_bounds) {
                if (e == hipSuccess) e = dev_alloc(&p->bounds, heads * 2 * head_dim);
                if (e == hipSuccess) e = dev_alloc(&p->scales, heads * 4);
                if (e == hipSuccess) e = hipMemset(p->bounds, 0, heads * 2 * head_dim);
                if (e == hipSuccess) e = hipMemset(p->scales, 0, heads * 4);
            }
        }
        if (e == hipSuccess) e = dev_alloc(&p->qk_norm, (size_t)n_layers * 2 * head_dim * 4);
        if (e == hipSuccess) e = hipDeviceSynchronize();
        if (e != hipSuccess) {
            const int rc = hip_fail(nullptr, e, name);
            free_paged(p);
            return rc;
        }
        *out = p;
        return PQA_OK;
    });
}

extern "C" void pqa_paged_destroy(pqa_paged* p) { free_paged(p); }

extern "C" const char* pqa_paged_last_error(const pqa_paged* p) { return p ? p->err.c_str() : pqa_last_error(nullptr); }

extern "C" int pqa_paged_memory(pqa_paged* p, void** key_pages, void** val_pages, int8_t** key_bounds, float** key_scales) {
    if (!p) return set_err(nullptr, PQA_ERR_ARG, "pqa_paged_memory: handle is NULL");
    if (key_pages) *key_pages = p->k;
    if (val_pages) *val_pages = p->v;
    if (key_bounds) *key_bounds = p->bounds;
    if (key_scales) *key_scales = p->scales;
    return PQA_OK;
}

extern "C" int pqa_paged_set_rope(pqa_paged* p, int rope_style, int rot_dim, int max_pos, const float* rope_cos,
                                  const float* rope_sin) {
    static const char* fn = "pqa_paged_set_rope";
    return guarded(p, fn, [&]() -> int {
        const std::string name = fn;
        if (!p) return fail(nullptr, PQA_ERR_ARG, name + ": handle is NULL");
        if (rot_dim < 0 || rot_dim > p->head_dim || rot_dim % 2)
            return fail(p, PQA_ERR_ARG, name + ": rot_dim must be even, from 0 to head_dim");
        if (rot_dim && (rope_style < 0 || rope_style > 2)) return fail(p, PQA_ERR_ARG, name + ": bad rope_style");
        if (rot_dim && max_pos <= 0) return fail(p, PQA_ERR_ARG, name + ": max_pos must be positive");
        if (rot_dim && (!rope_cos || !rope_sin)) return fail(p, PQA_ERR_ARG, name + ": RoPE tables are NULL");
        if (p->append_captured)
            return fail(p, PQA_ERR_ARG, name + ": a captured append holds the present tables");
        OnDevice on(p->device);
        if (on.err != hipSuccess) return hip_fail(p, on.err, name);
        float* tab = nullptr;
        if (rot_dim) {
            const size_t n = (size_t)max_pos * (rot_dim / 2) * 4;
            hipError_t e = dev_alloc(&tab, 2 * n);
            if (e == hipSuccess) e = hipMemcpy(tab, rope_cos, n, hipMemcpyHostToDevice);
            if (e == hipSuccess) e = hipMemcpy((char*)tab + n, rope_sin, n, hipMemcpyHostToDevice);
            if (e != hipSuccess) {
                if (tab) (void)hipFree(tab);
                return hip_fail(p, e, name);
            }
        }
        const hipError_t e = hipDeviceSynchronize();  // calls that still read the old tables
        if (e != hipSuccess) {
            if (tab) (void)hipFree(tab);
            return hip_fail(p, e, name);
        }
        if (p->rope) (void)hipFree(p->rope);
        p->rope = tab;
        p->rope_style = rope_style;
        p->rot_dim = rot_dim;
        p->max_pos = rot_dim ? max_pos : 0;
        return PQA_OK;
    });
}

extern "C" int pqa_paged_set_qk_norm(pqa_paged* p, int layer, const float* q_norm_w, const float* k_norm_w) {
    static const char* fn = "pqa_paged_set_qk_norm";
    return guarded(p, fn, [&]() -> int {
        const std::string name = fn;
        if (!p) return fail(nullptr, PQA_ERR_ARG, name + ": handle is NULL");
        if (layer < 0 || layer >= p->n_layers) return fail(p, PQA_ERR_ARG, name + ": layer out of range");
        if (!q_norm_w != !k_norm_w) return fail(p, PQA_ERR_ARG, name + ": give both weights or neither");
        if (!q_norm_w) {
            p->has_qk_norm[layer] = 0;
            return PQA_OK;
        }
        OnDevice on(p->device);
        hipError_t e = on.err;
        const size_t n = (size_t)p->head_dim * 4;
        char* dst = (char*)p->qk_norm + (size_t)layer * 2 * n;
        if (e == hipSuccess) e = hipDeviceSynchronize();  // calls that still read the old weights
        if (e == hipSuccess) e = hipMemcpy(dst, q_norm_w, n, hipMemcpyHostToDevice);
        if (e == hipSuccess) e = hipMemcpy(dst + n, k_norm_w, n, hipMemcpyHostToDevice);
        if (e != hipSuccess) return hip_fail(p, e, name);
        p->has_qk_norm[layer] = 1;
        return PQA_OK;
    });
}

extern "C" int pqa_batch_create(pqa_paged* p, pqa_batch** out, int max_seqs, int max_tokens, int max_len) {
    static const char* fn = "pqa_batch_create";
    return guarded(p, fn, [&]() -> int {
        const std::string name = fn;
        if (!p) return fail(nullptr, PQA_ERR_ARG, name + ": handle is NULL");
        if (!out) return fail(p, PQA_ERR_ARG, name + ": out is NULL");
        *out = nullptr;
        if (max_seqs <= 0 || max_tokens <= 0 || max_len <= 0) return fail(p, PQA_ERR_ARG, name + ": sizes must be positive");
        if (max_len > (1 << 30)) return fail(p, PQA_ERR_UNSUPPORTED, name + ": max_len above 2^30");  // tiles are counted in 31 bits
        if ((long long)max_tokens * (p->n_heads + 2LL * p->n_kv) * 16 >= (1LL << 31) || max_seqs >= (1 << 24))
            return fail(p, PQA_ERR_UNSUPPORTED, name + ": batch too large");
        pqa_batch* b = new pqa_batch();
        b->p = p;
        b->device = p->device;
        pqa::PagedShape& s = b->shape;
        s.n_pages = p->n_pages;
        s.page_size = p->page_size;
        s.group = p->group;
        s.n_kv = p->n_kv;
        s.narrow_wgs = pqa::paged_narrow_wgs(p->head_dim, p->cu_count);
        s.wide_wgs = pqa::paged_wide_wgs(p->head_dim, p->cu_count);
        s.wide_rows = pqa::paged_wide_rows(p->type, p->head_dim);
        s.least_rows = pqa::paged_least_rows();
        s.wide_keys = pqa::paged_wide_keys(p->head_dim);
        s.key_bytes = 4 * p->head_dim;
        s.max_seqs = max_seqs;
        s.max_tokens = max_tokens;
        s.max_seq_pages = (int)(((long long)max_len + p->page_size - 1) / p->page_size);
        b->max_touched = std::min<size_t>((size_t)max_tokens, (size_t)2 * max_seqs + max_tokens / p->page_size);
        b->max_rest = (size_t)max_seqs * p->n_kv + s.narrow_wgs;
        // blocks of every sequence (up to two of least_rows each, while these are fewer than wide_wgs), and their parts
        b->max_wide = ((size_t)max_tokens * p->group / s.wide_rows + max_seqs) * p->n_kv + 4 * s.wide_wgs;
        const size_t entries = (size_t)max_seqs * s.max_seq_pages;
        // no plan of this capacity leaves more partials: a block of rows is cut into at most max_len / kWideLeast + 1 parts
        const size_t rows = (size_t)max_tokens * p->group;
        const size_t blocks = rows <= pqa::kNarrowRows ? 0 : rows / s.least_rows + std::min(max_seqs, max_tokens);
        const size_t wide_parts = std::min<size_t>(pqa::paged_wide_slots(s), blocks * p->n_kv * ((size_t)max_len / pqa::kWideLeast + 1));
        struct {
            void** p;
            size_t bytes;
        } parts[] = {{(void**)&b->header, pqa::kPagedHeader * 4},
                     {(void**)&b->runs, (size_t)s.narrow_wgs * sizeof(pqa::PagedRun)},
                     {(void**)&b->rest, b->max_rest * sizeof(pqa::PagedItem)},
                     {(void**)&b->tokens, (size_t)max_tokens * sizeof(pqa::PagedToken)},
                     {(void**)&b->wide, b->max_wide * sizeof(pqa::PagedItem)},
                     {(void**)&b->touched, b->max_touched * sizeof(pqa::PagedTouched)},
                     {(void**)&b->pages, entries * 4},
                     {(void**)&b->counters, ((size_t)s.narrow_wgs + s.wide_wgs) * 4},
                     {(void**)&b->part_narrow, (size_t)pqa::paged_narrow_slots(s) * 16 * (p->head_dim + 2) * 4},
                     {(void**)&b->part_wide, wide_parts * s.wide_rows * (p->head_dim + 2) * 4}};
        size_t bytes = 0;
        for (const auto& q : parts) bytes += (q.bytes + 255) & ~(size_t)255;
        OnDevice on(p->device);
        hipError_t e = on.err;
        if (e == hipSuccess) e = dev_alloc(&b->mem, bytes);
        for (int i = 0; i < 2 && e == hipSuccess; i++) e = hipEventCreateWithFlags(&b->copied[i], hipEventDisableTiming);
        if (e == hipSuccess) {
            size_t off = 0;
            for (const auto& q : parts) {
                *q.p = b->mem + off;
                off += (q.bytes + 255) & ~(size_t)255;
            }
            e = hipMemset(b->mem, 0, (char*)b->part_narrow - b->mem);
        }
        if (e == hipSuccess) e = hipDeviceSynchronize();
        if (e != hipSuccess) {
            const int rc = hip_fail(p, e, name);
            free_batch(b);
            return rc;
        }
        *out = b;
        return PQA_OK;
    });
}

extern "C" void pqa_batch_destroy(pqa_batch* b) { free_batch(b); }

extern "C" int pqa_batch_set(pqa_batch* b, int n_seqs, const int* n_new, const int* len, const int* pages, int stride,
                             void* stream) {
    static const char* fn = "pqa_batch_set";
    return guarded(b ? b->p : nullptr, fn, [&]() -> int {
        const std::string name = fn;
        if (!b) return fail(nullptr, PQA_ERR_ARG, name + ": batch is NULL");
        pqa_paged* p = b->p;
        pqa::PagedShape s = b->shape;
        s.max_pos = p->max_pos;  // kept with the plan that was checked against it
        if (stride < 0) return fail(p, PQA_ERR_ARG, name + ": stride is negative");
        // a new plan beside the old one, which stays as it is if anything is wrong
        pqa::PagedPlan plan;
        std::string why;
        const PagedFault f = pqa::paged_check(s, n_seqs, n_new, len, pages, stride, &plan, &why);
        if (f != PagedFault::none) return fail(p, f == PagedFault::range ? PQA_ERR_RANGE : PQA_ERR_ARG, name + ": " + why);
        pqa::paged_items(s, &plan);
        if (plan.runs.size() > (size_t)s.narrow_wgs || plan.rest.size() > b->max_rest || plan.wide.size() > b->max_wide ||
            plan.touched.size() > b->max_touched)
            return fail(p, PQA_ERR_ARG, name + ": plan exceeds the batch");  // cannot happen: the capacities follow from the checks
        OnDevice on(b->device);
        hipStream_t st = (hipStream_t)stream;
        bool captured = false;
        hipError_t e = on.err;
        if (e == hipSuccess) e = is_captured(st, &captured);
        if (e != hipSuccess) return hip_fail(p, e, name);
        if (captured) return fail(p, PQA_ERR_ARG, name + ": not while the stream is captured (replayed calls follow a later set)");
        const bool small = plan.wide_rows < s.wide_rows;
        const int header[pqa::kPagedHeader] = {plan.n_tok, (int)plan.touched.size(), (int)plan.runs.size(),
                                               small ? 0 : (int)plan.wide.size(), small ? (int)plan.wide.size() : 0};
        const struct {
            void* dst;
            const void* src;
            size_t bytes;
        } parts[] = {{b->header, header, sizeof header},
                     {b->runs, plan.runs.data(), plan.runs.size() * sizeof(pqa::PagedRun)},
                     {b->rest, plan.rest.data(), plan.rest.size() * sizeof(pqa::PagedItem)},
                     {b->tokens, plan.tokens.data(), plan.tokens.size() * sizeof(pqa::PagedToken)},
                     {b->wide, plan.wide.data(), plan.wide.size() * sizeof(pqa::PagedItem)},
                     {b->touched, plan.touched.data(), plan.touched.size() * sizeof(pqa::PagedTouched)},
                     {b->pages, plan.pages.data(), plan.pages.size() * 4}};
        // One copy of the tables from the first to the last byte in use where that is little more
        // than what is used (a copy costs some 5 us whatever its size), else one for each.
        const size_t span = (size_t)((char*)b->pages + plan.pages.size() * 4 - b->mem);
        size_t used = 0;
        for (const auto& q : parts) used += (q.bytes + 15) & ~(size_t)15;
        const bool whole = span <= used + (64 << 10);
        const size_t need = whole ? span : used;
        const int turn = b->turn;
        if (b->stage_bytes[turn] < need) {
            e = hipEventSynchronize(b->copied[turn]);
            if (e == hipSuccess && b->stage[turn]) e = hipHostFree(b->stage[turn]);
            b->stage[turn] = nullptr;
            b->stage_bytes[turn] = 0;
            const size_t room = std::max<size_t>(need + need / 2, 64 << 10);
            if (e == hipSuccess) e = hipHostMalloc((void**)&b->stage[turn], room, hipHostMallocDefault);
            if (e != hipSuccess) return hip_fail(p, e, name);
            std::memset(b->stage[turn], 0, room);
            b->stage_bytes[turn] = room;
        } else if ((e = hipEventSynchronize(b->copied[turn])) != hipSuccess) {  // the copy before last has left the buffer
            return hip_fail(p, e, name);
        }
        // from here on the tables change: nothing may run with a plan that is half there
        b->set = false;
        char* stage = b->stage[turn];
        size_t off = 0;
        for (const auto& q : parts) {
            if (!q.bytes) continue;
            char* at = whole ? stage + ((char*)q.dst - b->mem) : stage + off;
            std::memcpy(at, q.src, q.bytes);
            if (!whole && e == hipSuccess) e = hipMemcpyAsync(q.dst, at, q.bytes, hipMemcpyHostToDevice, st);
            off += (q.bytes + 15) & ~(size_t)15;
        }
        if (whole && e == hipSuccess) e = hipMemcpyAsync(b->mem, stage, span, hipMemcpyHostToDevice, st);
        if (e == hipSuccess) e = hipEventRecord(b->copied[turn], st);
        if (e != hipSuccess) return hip_fail(p, e, name);
        b->turn ^= 1;
        b->plan = std::move(plan);
        b->shape.max_pos = s.max_pos;
        b->set = true;
        return PQA_OK;
    });
}

namespace {

// What every call on a batch checks first. Sets *captured.
int begin(pqa_paged* p, pqa_batch* b, int layer, const OnDevice& on, void* stream, const char* fn, bool* captured) {
    const std::string name = fn;
    if (b->p != p) return fail(p, PQA_ERR_ARG, name + ": the batch belongs to another handle");
    if (layer < 0 || layer >= p->n_layers) return fail(p, PQA_ERR_ARG, name + ": layer out of range");
    if (!b->set) return fail(p, PQA_ERR_ARG, name + ": the batch holds nothing yet (pqa_batch_set)");
    hipError_t e = on.err;
    if (e == hipSuccess) e = is_captured((hipStream_t)stream, captured);
    return e == hipSuccess ? PQA_OK : hip_fail(p, e, name);
}

// Rows of at least `width` elements at distance ld, aligned to their elements.
int check_rows(pqa_paged* p, const void* rows, long long ld, int heads, const char* what, const char* fn) {
    if (!rows) return fail(p, PQA_ERR_ARG, std::string(fn) + ": " + what + " is NULL");
    if (ld < (long long)heads * p->head_dim)
        return fail(p, PQA_ERR_ARG, std::string(fn) + ": rows of " + what + " overlap (distance " + std::to_string(ld) + ")");
    if ((uintptr_t)rows % pqa::paged_io_bytes(p->type))
        return fail(p, PQA_ERR_ARG, std::string(fn) + ": " + what + " is misaligned");
    return PQA_OK;
}

int append(pqa_paged* p, pqa_batch* b, int layer, const pqa::PagedRows& q, const pqa::PagedRows& k, const pqa::PagedRows& v,
           void* q_out, long long ldo, bool captured, hipStream_t s, const char* fn) {
    if (!b->plan.n_tok && !captured) return PQA_OK;
    if (int rc = check_rows(p, q.p, q.ld, p->n_heads, "q", fn)) return rc;
    if (int rc = check_rows(p, k.p, k.ld, p->n_kv, "k", fn)) return rc;
    if (int rc = check_rows(p, v.p, v.ld, p->n_kv, "v", fn)) return rc;
    if (int rc = check_rows(p, q_out, ldo, p->n_heads, "the output", fn)) return rc;
    if (p->max_pos != b->shape.max_pos)
        return fail(p, PQA_ERR_ARG, std::string(fn) + ": the rotation changed after pqa_batch_set; set the batch again");
    if (captured) p->append_captured = true;
    const hipError_t e = pqa::launch_paged_append(b, layer, q, k, v, q_out, ldo, captured, s);
    return e == hipSuccess ? PQA_OK : hip_fail(p, e, fn);
}

int attend(pqa_paged* p, pqa_batch* b, int layer, const pqa::PagedRows& q, void* out, long long ldo, bool captured, hipStream_t s,
           const char* fn) {
    if (!b->plan.n_tok && !captured) return PQA_OK;
    if (int rc = check_rows(p, q.p, q.ld, p->n_heads, "q", fn)) return rc;
    if (int rc = check_rows(p, out, ldo, p->n_heads, "out", fn)) return rc;
    const hipError_t e = pqa::launch_paged_attend(b, layer, q, out, ldo, captured, s);
    return e == hipSuccess ? PQA_OK : hip_fail(p, e, fn);
}

}  // namespace

extern "C" int pqa_paged_append(pqa_paged* p, pqa_batch* b, int layer, const void* q, int64_t q_stride, const void* k,
                                int64_t k_stride, const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride,
                                void* stream) {
    static const char* fn = "pqa_paged_append";
    return guarded(p, fn, [&]() -> int {
        if (!p || !b) return fail(p, PQA_ERR_ARG, std::string(fn) + ": handle or batch is NULL");
        OnDevice on(p->device);
        bool captured = false;
        if (int rc = begin(p, b, layer, on, stream, fn, &captured)) return rc;
        return append(p, b, layer, {q, q_stride}, {k, k_stride}, {v, v_stride}, q_out, q_out_stride, captured, (hipStream_t)stream, fn);
    });
}

extern "C" int pqa_paged_attend(pqa_paged* p, pqa_batch* b, int layer, const void* q, int64_t q_stride, void* out,
                                int64_t out_stride, void* stream) {
    static const char* fn = "pqa_paged_attend";
    return guarded(p, fn, [&]() -> int {
        if (!p || !b) return fail(p, PQA_ERR_ARG, std::string(fn) + ": handle or batch is NULL");
        OnDevice on(p->device);
        bool captured = false;
        if (int rc = begin(p, b, layer, on, stream, fn, &captured)) return rc;
        return attend(p, b, layer, {q, q_stride}, out, out_stride, captured, (hipStream_t)stream, fn);
    });
}

extern "C" int pqa_paged_forward(pqa_paged* p, pqa_batch* b, int layer, const void* q, int64_t q_stride, const void* k,
                                 int64_t k_stride, const void* v, int64_t v_stride, void* out, int64_t out_stride, void* stream) {
    static const char* fn = "pqa_paged_forward";
    return guarded(p, fn, [&]() -> int {
        if (!p || !b) return fail(p, PQA_ERR_ARG, std::string(fn) + ": handle or batch is NULL");
        OnDevice on(p->device);
        bool captured = false;
        if (int rc = begin(p, b, layer, on, stream, fn, &captured)) return rc;
        // q normed and rotated passes through the output rows
        if (int rc = append(p, b, layer, {q, q_stride}, {k, k_stride}, {v, v_stride}, out, out_stride, captured, (hipStream_t)stream, fn))
            return rc;
        return attend(p, b, layer, {out, out_stride}, out, out_stride, captured, (hipStream_t)stream, fn);
    });
}

extern "C" int pqa_paged_attend_sparse(pqa_paged* p, pqa_batch* b, int layer, const void* q, int64_t q_stride, int select,
                                       int first, int last, int* chosen, void* out, int64_t out_stride, void* stream) {
    static const char* fn = "pqa_paged_attend_sparse";
    return guarded(p, fn, [&]() -> int {
        const std::string name = fn;
        if (!p || !b) return fail(p, PQA_ERR_ARG, name + ": handle or batch is NULL");
        OnDevice on(p->device);
        bool captured = false;
        if (int rc = begin(p, b, layer, on, stream, fn, &captured)) return rc;
        if (!p->bounds) return fail(p, PQA_ERR_ARG, name + ": the handle was created without key bounds");
        if (select < 1 || first < 0 || last < 1 || (long long)first + last > select)
            return fail(p, PQA_ERR_ARG, name + ": need first >= 0, last >= 1 and first + last <= select");
        if ((long long)select * p->page_size >= (1LL << 31) || (long long)b->shape.max_tokens * p->n_kv * select >= (1LL << 40))
            return fail(p, PQA_ERR_UNSUPPORTED, name + ": select is too large");
        if (!b->plan.n_tok && !captured) return PQA_OK;
        if (!chosen || (uintptr_t)chosen & 3u) return fail(p, PQA_ERR_ARG, name + ": chosen is NULL or misaligned");
        if (int rc = check_rows(p, q, q_stride, p->n_heads, "q", fn)) return rc;
        if (int rc = check_rows(p, out, out_stride, p->n_heads, "out", fn)) return rc;
        int longest = captured ? b->shape.max_seq_pages : 0;
        for (const pqa::PagedSeq& s : b->plan.seqs)
            if (s.n_new) longest = std::max(longest, (s.len + p->page_size - 1) / p->page_size);
        if (longest > pqa::kPagedMaxChoice)
            return fail(p, PQA_ERR_UNSUPPORTED, name + ": more than " + std::to_string(pqa::kPagedMaxChoice) +
                                                    " pages in a sequence" + (captured ? " (captured: the batch's most)" : ""));
        const pqa::PagedRows rows = {q, q_stride};
        const hipError_t e =
            pqa::launch_paged_sparse(b, layer, rows, select, first, last, chosen, out, out_stride, captured, (hipStream_t)stream);
        return e == hipSuccess ? PQA_OK : hip_fail(p, e, name);
    });
}
