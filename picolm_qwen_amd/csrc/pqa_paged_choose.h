// The choice of pages, shared by the kernels that make it alone (pqa_paged_choose.hip) and with the
// attention after it (pqa_paged_attn.hip).
//
// Which pages a query token attends to under a page budget: per KV head the `first` pages, the
// `last` ones that end with the token's own, and those of the largest scores,
//   score(page) = 2^(e_page - 6) max_h 2^(e_h - 6) sum_d max(q_hd lo_d, q_hd hi_d),
// with the page's key bounds lo, hi and the query head's row q_h as whole numbers of 7 bits and a
// sign: (nearly) the largest logit that a key of the page can have. With q split by sign the sum
// is one product of [min(q, 0), max(q, 0)] with [lo, hi] on the int8 matrix instructions, 16 pages
// by 16 heads at a time; it is a whole number below 2^22 and the scales are powers of two, so
// every score is exact and the choice is the same in any order of summation.
//
// A workgroup takes a KV head of one token, or of as many tokens of a chunk as fill the 16 columns
// of a product (they share each page's bounds): scores to LDS as integers in the floats' order, then per token
// the least chosen key and the list in ascending order (the lower page where scores are equal). Up to
// kWaveKeys pages a wave keeps a token's keys in registers and finds that key bit by bit,
// counting by ballots (no barrier); longer lists go through the whole workgroup, by digits.
// Bound by reading the bounds, 2 head_dim + 4 bytes per page and KV head, and for single tokens
// by the latency of that.
#pragma once

#include "pqa_paged_device.h"

namespace pqa {

typedef int intx4 __attribute__((ext_vector_type(4)));

struct PagedChoose {
    const void* q;
    long long ldq;
    const int8_t* bounds;  // the layer's
    const float* scales;
    const int* header;
    const int* tokens;  // PagedToken
    const int* pages;
    int* chosen;
    int g, n_kv, shift, select, first, last, qvec;
    int group, stride;  // tokens per workgroup; keys per token in LDS
    int single;         // no sequence has more than one new token
    int parts;          // workgroups that share a column's pages (group 1)
    uint32_t* part_keys;  // [column][stride]
    unsigned* counters;
};

// Threads: 1024 for single tokens, whose few workgroups wait for loads; 512 where tokens share one, and at
// head sizes whose operands need the registers.
template <int HD>
constexpr int choose_threads() { return HD <= 128 ? 1024 : 512; }
constexpr int kChooseWaves = 16;
constexpr int kWaveKeys = 1024;
constexpr int kPartPages = 512;  // least pages of a column's part
constexpr int kChooseBytes = 40 << 10;  // of LDS for the keys, where more than one token shares a workgroup

// 16 elements as whole numbers, rounded to nearest even, of one sign within [lo, hi] and the others as
// zero: past 3 * 2^22 a float's step is one, and its low byte the number in two's complement
__device__ __forceinline__ intx4 signed_bytes(const float (&x)[16], float up, float lo, float hi) {
    intx4 out;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        unsigned b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) b[e] = __float_as_uint(__builtin_amdgcn_fmed3f(x[4 * w + e] * up, lo, hi) + 12582912.0f);
        const unsigned ab = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), cd = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
        out[w] = (int)(ab | cd);
    }
    return out;
}

// a float as an unsigned integer of the same order
__device__ __forceinline__ uint32_t ordered_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int popcount(unsigned long long x) { return (int)__popcll(x); }

// bits of x below the lane's
__device__ __forceinline__ int before(unsigned long long x) {
    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(x >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)x, 0));
}

// A token's keys: its forced pages, [0, first) and [p1, n), above all scores.
struct Keys {
    const uint32_t* k;
    int first, p1, n;
    __device__ uint32_t operator[](int i) const { return i < first || i >= p1 ? 0xFFFFFFFFu : k[i]; }
};

// maximum over the wave's lanes, in every lane
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor1, 0xF, 0xF, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor2, 0xF, 0xF, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor7, 0xF, 0xF, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor15, 0xF, 0xF, false));
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max((uint32_t)b[0], (uint32_t)b[1]);
}

// The list of one token by one wave, its n <= 64 R keys in registers.
template <int R>
__device__ __forceinline__ void choose_by_wave(const Keys& keys, int select, int lane, int* out) {
    uint32_t k[R], hi = 0, lo = 0;  // lo: of the complements
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = 64 * r + lane;
        const uint32_t x = i < keys.n ? keys.k[i] : 0u;
        const bool score = i >= keys.first && i < keys.p1;
        if (score) {
            hi = max(hi, x);
            lo = max(lo, ~x);
        }
        k[r] = i >= keys.n ? 0u : score ? x : 0xFFFFFFFFu;
    }
    hi = __builtin_amdgcn_readfirstlane(wave_max(hi));
    lo = __builtin_amdgcn_readfirstlane(~wave_max(lo));
    auto count = [&](uint32_t least) {
        int c = 0;
#pragma unroll
        for (int r = 0; r < R; r++) c += popcount(__ballot(k[r] >= least));
        return c;
    };
    // the largest key that at least `select` keys reach, from the highest bit on in which two scores
    // differ (the forced pages' keys are above all of them)
    const int top = lo == hi ? -1 : 31 - __clz((int)(lo ^ hi));
    uint32_t least = top < 0 ? lo : top == 31 ? 0u : lo >> (top + 1) << (top + 1);
    int reach = top == 31 ? keys.n : count(least);
#pragma unroll 1
    for (int bit = top; bit >= 0 && reach != select; bit--) {
        const uint32_t cand = least | 1u << bit;
        const int c = count(cand);
        if (c >= select) {
            least = cand;
            reach = c;
        }
    }
    // above it all, of those that equal it the first `same`
    int same = reach == select ? keys.n : select - (least == 0xFFFFFFFFu ? 0 : count(least + 1)), put = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool in = 64 * r + lane < keys.n, is = in && k[r] == least;
        const unsigned long long equal = __ballot(is);
        const bool take = in && (k[r] > least || (is && before(equal) < same));
        const unsigned long long taken = __ballot(take);
        const int to = put + before(taken);
        if (take && to < select) out[to] = 64 * r + lane;
        put += popcount(taken);
        same = max(0, same - popcount(equal));
    }
}

// What the listing of a long column by a workgroup needs of LDS.
struct ListScratch {
    int hist[256];
    uint32_t lo[kChooseWaves], hi[kChooseWaves];
    int gt[kChooseWaves], eq[kChooseWaves];
    int digit, left;
};

// Scores of pages [p0, p1) for nt tokens from tok on, to keys[token * stride + page], which are 0 elsewhere; by the
// whole workgroup (waves w of `waves`), which has to wait for each other afterwards. 16 columns of a product: the
// heads of the tokens, or 16 heads at a time. PB: blocks of 16 pages at a time.
template <int TYPE, int HD, int PB>
__device__ __forceinline__ void score_pages(const PagedChoose& a, uint32_t* keys, int tok, int nt, int kvh, int table, int p0,
                                            int p1, int w, int waves) {
    typedef typename PagedType<TYPE>::Io Io;
    constexpr int ST = HD / 32;  // steps of 64 products
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, c16 = lane & 15, g16 = lane >> 4;
    bool ready = false;
    for (int h0 = 0; h0 < a.g; h0 += 16) {
        const int t = a.g > 16 ? 0 : c16 / a.g, h = a.g > 16 ? h0 + c16 : c16 - t * a.g;
        const bool column = t < nt && h < a.g;  // the others repeat column 0
        const Io* q = (const Io*)a.q + (long long)(column ? tok + t : tok) * a.ldq + (long long)(kvh * a.g + (column ? h : 0)) * HD;
        int page[PB];
        auto look = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < PB; b++) page[b] = a.pages[table + min(b0 + 16 * b + c16, p1 - 1)];
        };
        int b0 = p0 + 16 * PB * w;
        if (b0 < p1) look(b0);
        float x[ST][16], mx = 0.0f;
#pragma unroll
        for (int st = 0; st < ST; st++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 y = load4(q + 16 * ((4 * st + g16) % (HD / 16)) + 4 * i, a.qvec);
                x[st][4 * i] = y.x;
                x[st][4 * i + 1] = y.y;
                x[st][4 * i + 2] = y.z;
                x[st][4 * i + 3] = y.w;
            }
        if (!ready) {  // the keys start below all scores; q's loads are on their way meanwhile
            for (int i = tid; i < nt * a.stride; i += threads) keys[i] = 0u;
            __syncthreads();
            ready = true;
        }
#pragma unroll
        for (int st = 0; st < ST; st++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, fabsf(x[st][i]));
        const int e = bound_exponent(max_x32(max_x16(mx)));
        const float up = power2(6 - e), down = power2(e - 6);
        intx4 qb[ST];
#pragma unroll
        for (int st = 0; st < ST; st++) {
            const bool neg = 4 * st + g16 < HD / 16;
            qb[st] = signed_bytes(x[st], up, neg ? -127.0f : 0.0f, neg ? 0.0f : 127.0f);
        }
        uint32_t* mine = keys + (column ? t : 0) * a.stride;
        for (; b0 < p1; b0 += 16 * PB * waves) {
            intx4 y[PB][ST];
            float sc[PB];
#pragma unroll
            for (int b = 0; b < PB; b++) {
                const size_t at = (size_t)page[b] * a.n_kv + kvh;
                const int8_t* r = a.bounds + at * (2 * HD) + 16 * g16;
#pragma unroll
                for (int st = 0; st < ST; st++) y[b][st] = *(const intx4*)(r + 64 * st);
                sc[b] = a.scales[at];  // of page b0 + 16 b + c16
            }
            if (b0 + 16 * PB * waves < p1) look(b0 + 16 * PB * waves);
#pragma unroll
            for (int b = 0; b < PB; b++) {
                intx4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int st = 0; st < ST; st++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[b][st], qb[st], acc, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; j++) {  // page 4 g16 + j of column c16
                    const float s = (float)acc[j] * down * __shfl(sc[b], 4 * g16 + j);
                    const int i = b0 + 16 * b + 4 * g16 + j;
                    if (column && i < p1) atomicMax(mine + i, min(ordered_bits(s), 0xFFFFFFFEu));
                }
            }
        }
    }
}

// The list of one token by the whole workgroup.
__device__ __forceinline__ void choose_by_block(const Keys& keys, int select, ListScratch& s, int w, int waves, int* out) {
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, n = keys.n, p0 = keys.first, p1 = keys.p1;
    // the range of the scores, so that the first digit tells them apart
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    for (int i = p0 + tid; i < p1; i += threads) {
        lo = min(lo, keys.k[i]);
        hi = max(hi, keys.k[i]);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
    }
    if (lane == 0) {
        s.lo[w] = lo;
        s.hi[w] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < waves; i++) {
        lo = min(lo, s.lo[i]);
        hi = max(hi, s.hi[i]);
    }
    // the `left`-th largest of keys [p0, p1) by digits of 8 bits of key - lo, from the top:
    // key - lo has `bits` bits, of which those above `shift` are known to be `prefix`
    const int bits = hi > lo ? 32 - __clz((int)(hi - lo)) : 0;
    int left = select - (n - (p1 - p0));
    uint32_t prefix = 0;
    int shift = bits;
    if (left > 0)
        while (shift > 0) {
            const int width = min(8, shift), next = shift - width;
            for (int i = tid; i < 256; i += threads) s.hist[i] = 0;
            __syncthreads();
            for (int i = p0 + tid; i < p1; i += threads) {
                const uint32_t k = keys.k[i] - lo;
                if (shift >= 32 || (k >> shift) == prefix) atomicAdd(&s.hist[(k >> next) & ((1u << width) - 1)], 1);
            }
            __syncthreads();
            if (w == 0) {  // lane l: digits 4 l .. 4 l + 3; the sum of all larger ones by a scan
                int c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) sum += c[j] = s.hist[4 * lane + j];
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
                        s.digit = 4 * lane + j;
                        s.left = left - over;
                    }
                    over += c[j];
                }
            }
            __syncthreads();
            prefix = prefix << width | (uint32_t)s.digit;
            left = s.left;
            shift = next;
        }
    // keys above lo + prefix are chosen, and the first `left` that equal it (left == 0: the
    // forced pages alone); each wave lists a run of the pages behind what the waves before it found
    const uint32_t at = left > 0 ? lo + prefix : 0xFFFFFFFEu;
    const int run = (n + waves * 64 - 1) / (waves * 64) * 64, r0 = w * run, r1 = min(n, r0 + run);
    int gt = 0, eq = 0;
    for (int i = r0 + lane; i < r1; i += 64) {
        const uint32_t k = keys[i];
        gt += k > at;
        eq += k == at;
    }
    for (int d = 32; d; d >>= 1) {
        gt += __shfl_xor(gt, d);
        eq += __shfl_xor(eq, d);
    }
    if (lane == 0) {
        s.gt[w] = gt;
        s.eq[w] = eq;
    }
    __syncthreads();
    int put = 0, same = 0;  // listed, and equal ones met, before this wave's run
    for (int i = 0; i < w; i++) {
        put += s.gt[i] + min(s.eq[i], max(0, left - same));
        same += s.eq[i];
    }
    const unsigned long long below = (1ull << lane) - 1;
    for (int i0 = r0; i0 < r1; i0 += 64) {
        const int i = i0 + lane;
        const uint32_t k = i < r1 ? keys[i] : 0u;
        const bool is = i < r1 && k == at;
        const unsigned long long equal = __ballot(is);
        const bool take = i < r1 && (k > at || (is && same + popcount(equal & below) < left));
        const unsigned long long taken = __ballot(take);
        const int to = put + popcount(taken & below);
        if (take && to < select) out[to] = i;
        put += popcount(taken);
        same += popcount(equal);
    }
    __syncthreads();
}

// host side (pqa_paged_choose.hip)
PagedChoose choose_arguments(const pqa_batch* b, int layer, const PagedRows& q, int select, int first, int last, int* chosen,
                             bool captured);
hipError_t launch_paged_choose(const pqa_batch* b, const PagedChoose& a, bool captured, hipStream_t s);

}  // namespace pqa
