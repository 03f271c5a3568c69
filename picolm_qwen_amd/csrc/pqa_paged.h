// The paged cache's handle, its batches and the launchers of its kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <string>
#include <vector>

#include "pqa.h"
#include "pqa_paged_plan.h"

struct pqa_paged {
    int n_layers = 0, n_pages = 0, page_size = 0, page_shift = 0, n_heads = 0, n_kv = 0, head_dim = 0, group = 1;
    int type = 0;
    bool owned = false;
    char* k = nullptr;  // [n_layers][n_pages][n_kv][page_size][head_dim], 2 bytes each
    char* v = nullptr;
    int8_t* bounds = nullptr;  // [n_layers][n_pages][n_kv][2][head_dim], or null
    float* scales = nullptr;   // [n_layers][n_pages][n_kv]
    size_t layer_bytes = 0;    // of K, and of V
    size_t layer_heads = 0;    // n_pages * n_kv

    int rope_style = 0, rot_dim = 0, max_pos = 0;
    float* rope = nullptr;  // cos then sin, [max_pos][rot_dim / 2] each
    float* qk_norm = nullptr;  // [n_layers][2][head_dim]
    std::vector<char> has_qk_norm;
    bool append_captured = false;  // a graph holds the address of the tables

    int cu_count = 256, device = 0;
    std::string err;
};

struct pqa_batch {
    pqa_paged* p = nullptr;
    int device = 0;
    pqa::PagedShape shape{};
    pqa::PagedPlan plan;
    bool set = false;
    // one device allocation: the tables below, then the partial results
    char* mem = nullptr;
    int* header = nullptr;  // kPagedHeader ints
    pqa::PagedToken* tokens = nullptr;
    int* pages = nullptr;
    pqa::PagedTouched* touched = nullptr;
    pqa::PagedRun* runs = nullptr;
    pqa::PagedItem* rest = nullptr;
    pqa::PagedItem* wide = nullptr;
    unsigned* counters = nullptr;  // zero between calls: narrow_wgs, then wide_wgs
    float* part_narrow = nullptr;
    float* part_wide = nullptr;
    size_t max_touched = 0, max_rest = 0, max_wide = 0;
    // two pinned staging buffers in turn, so that a set waits for the copy before last
    char* stage[2] = {nullptr, nullptr};
    size_t stage_bytes[2] = {0, 0};
    hipEvent_t copied[2] = {nullptr, nullptr};
    int turn = 0;
};

namespace pqa {

// what the kernels read of a batch, so that a captured call follows the batch's later sets
enum : int { kHdTokens = 0, kHdTouched = 1, kHdRuns = 2, kHdWide = 3, kHdSmall = 4, kPagedHeader = 8 };

inline bool paged_head_dim(int hd) { return hd == 64 || hd == 96 || hd == 128 || hd == 160 || hd == 192 || hd == 256; }
inline int paged_io_bytes(int type) { return type == PQA_PAGED_F32 ? 4 : 2; }

// the attention kernels' tiles (pqa_paged_attn.hip)
int paged_wide_rows(int type, int hd);
int paged_least_rows();
int paged_wide_keys(int hd);
int paged_narrow_wgs(int hd, int cu_count);
int paged_wide_wgs(int hd, int cu_count);

struct PagedRows {  // token rows: base and distance in elements
    const void* p;
    long long ld;
};

hipError_t launch_paged_append(const pqa_batch* b, int layer, const PagedRows& q, const PagedRows& k, const PagedRows& v,
                               void* q_out, long long ldo, bool captured, hipStream_t s);
hipError_t launch_paged_attend(const pqa_batch* b, int layer, const PagedRows& q, void* out, long long ldo, bool captured,
                               hipStream_t s);
// most pages of one sequence that a choice can be made of: their scores fit the LDS
constexpr int kPagedMaxChoice = 32768;
hipError_t launch_paged_sparse(const pqa_batch* b, int layer, const PagedRows& q, int select, int first, int last, int* chosen,
                               void* out, long long ldo, bool captured, hipStream_t s);

}  // namespace pqa
