// Attention of a batch's new tokens over their sequences' pages:
//   out = sum_j 2^(s_j - M) v_j / sum_j 2^(s_j - M),  s_j = (q . k_j) log2(e) / sqrt(d),
// over the keys j up to the token's own position, in one pass with a running maximum M.
//
// Rows (query heads of one KV head, token by token) are packed 16 to a tile column:
// S^T = K Q^T and O^T += V^T P^T on 16x16x32 matrix instructions, in whose layouts a lane's
// scores are already its operand of the second product. Keys lie in blocks of 16, each within
// one page ([page][kv_head][row][dim]) and so contiguous in memory; they arrive by direct
// global->LDS loads, 16-byte chunk c of row r at slot c ^ x(r), which keeps the K operand reads
// and the transposing V reads free of bank conflicts.
//
// Types: fp16 and bf16 rows enter the products as they are. P is rounded to the same type in the wide
// kernel (half a step, 2^-11 or 2^-8 of a weight, which leaves at most as much error as the output's
// own rounding; a second product would cost a third of its time), and split into a high and a low part in the narrow
// one, where products are free (not by the workgroups of two waves, which a chunk's chosen pages feed
// from the caches: 191 us with it, 178 without, for 300 tokens). fp32 rows are split into two fp16 parts with 22
// significant bits together (after an exact power of two), and so is P, the low parts' sums
// apart: fp32-level results at twice the products. Scores, maxima and sums are fp32 throughout.
//
// Two kernels:
//   narrow  up to 16 rows per sequence and KV head (single tokens): bound by reading K and V
//           once. Waves take 32-key tiles in turn, each with two tiles of its own in flight,
//           and meet in LDS. The batch's key tiles are cut into one run per workgroup, so
//           that contexts of any mix of lengths keep all of them busy to the end.
//   wide    more rows (chunks): bound by the products. 4 waves share each key tile (two
//           buffers, one barrier per tile).
// Rows whose keys were cut leave partial sums, which the last workgroup of these rows to
// finish joins in a fixed order (results do not depend on which one that is).
//
// Measured (one call after another, inputs changing): 48 tokens behind 345k positions, bf16, 32 / 8 heads of 128,
// 183 us (6.4 TB/s); one behind 131072, fp16, 90 us (6.0 TB/s); one behind 700, fp32, 14 / 2 heads of 64, 8.3 us
// (dependent loads); 2048 tokens behind 6000, bf16, 244 us (967 TFLOP/s; a large product of the
// library reaches 1240).
//
// A split product can turn inf into NaN (inf * 0, inf - inf), and a masked key's V row still
// enters the product with weight 0. A row whose result is not finite is therefore computed again by
// slow_rows, in fp32 over its own keys alone.
#include <algorithm>

#include "pqa_paged_choose.h"

namespace pqa {

namespace {

constexpr float kNone = -3.0e38f;  // running maximum before the first key
constexpr float kSlack = 4.0f;     // P is rescaled when a score passes the maximum by this many log2 units
constexpr float kLow = 2048.0f;    // scale of P's low parts, to the exponents of the high ones

struct PagedAttn {
    const void* q;
    void* out;
    long long ldq, ldo;
    const char* kp;  // the layer's pages
    const char* vp;
    const int* pages;
    const int* items;  // PagedItem: the wide ones, or those behind the runs' first
    const int* runs;   // PagedRun
    const int* header;
    float* part;
    unsigned* counters;
    const int* chosen;  // attention over chosen pages: [token][kv head][select], else null
    const int* tokens;  // PagedToken
    int select, wgs;
    int crowd;  // chosen pages of many columns: workgroups of two waves, so that two share a CU
    int g, n_kv, shift;
    int qvec, ovec;  // rows may move as 16-byte vectors
    float qscale;
};

// rows and keys of one piece of work
struct Column {
    int row0, rows, hist, table, kvh, r0;
    int kend;          // keys that exist
    const int* list;   // its chosen pages, or null: all pages of the sequence
    const int* local;  // in LDS: ids of the chosen pages themselves, or null
};

constexpr int pow2_of(int ch) { return ch % 16 == 0 ? 16 : ch % 8 == 0 ? 8 : ch % 4 == 0 ? 4 : ch % 2 == 0 ? 2 : 1; }

template <int HD>
struct Geo {
    static_assert(HD % 32 == 0 && HD <= 256, "whole 1 KB loads per block of 16 keys");
    static constexpr int CH = HD / 8;         // 16-byte chunks per row
    static constexpr int ROWB = HD * 2;
    static constexpr int BLKB = 16 * ROWB;    // a block of 16 keys
    static constexpr int PPB = BLKB / 1024;   // its 1 KB loads
    static constexpr int P2 = pow2_of(CH);
    static constexpr int PER = 16 / P2 > 0 ? 16 / P2 : 1;  // rows after which the bank of a chunk repeats
    static constexpr int KS = HD / 32, DB = HD / 16;
    static constexpr int QS = HD + 4;  // row stride of fp32 rows in LDS
    __device__ static int xk(int r) { return (r / PER) & (P2 - 1); }
    __device__ static int xv(int r) { return (2 * (r / PER)) & (P2 - 1); }
};

template <int TYPE>
struct Ops;
template <>
struct Ops<PQA_PAGED_F16> {
    typedef half8 V8;
    static constexpr bool split = false;
    static constexpr float scale = 2048.0f;  // of P: fp16's exponents reach down to 2^-25 of the largest weight
    __device__ static floatx4 mul(V8 a, V8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Ops<PQA_PAGED_F32> : Ops<PQA_PAGED_F16> {
    static constexpr bool split = true;
};
template <>
struct Ops<PQA_PAGED_BF16> {
    typedef bf16x8 V8;
    static constexpr bool split = false;
    static constexpr float scale = 1.0f;
    __device__ static floatx4 mul(V8 a, V8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ int page_at(const PagedAttn& a, const Column& c, int i) {
    if (c.local) return __builtin_amdgcn_readfirstlane(c.local[i]);
    const int j = c.list ? scalar_int(c.list, i) : i;
    return scalar_int(a.pages, c.table + j);
}

// byte offset of the block of 16 keys at `pos` in page `page`
template <int HD>
__device__ __forceinline__ size_t block_offset(const PagedAttn& a, const Column& c, int page, int pos) {
    return (size_t)((((unsigned)page * a.n_kv + c.kvh) << a.shift) + (pos & ((1 << a.shift) - 1))) * Geo<HD>::ROWB;
}

// element offset of packed row R in rows of distance ld
template <int HD>
__device__ __forceinline__ long long row_offset(const PagedAttn& a, const Column& c, int R, long long ld) {
    const int tok = R / a.g;
    return (long long)(c.row0 + tok) * ld + (c.kvh * a.g + R - tok * a.g) * HD;
}

// What a wave carries for one block of 16 rows; lane (c16, g16) holds row c16's.
template <int TYPE, int HD>
struct RowBlock {
    typedef typename Ops<TYPE>::V8 V8;
    static constexpr int KS = Geo<HD>::KS, DB = Geo<HD>::DB;
    static constexpr bool split = Ops<TYPE>::split;
    V8 q[KS], ql[split ? KS : 1];  // dims 32 ks + 8 g16 .. +7; high and low parts
    float cs;                      // a raw score's factor to log2 units
    int qpos;
    float m, l;  // the maximum of the raw scores, and the lane's share of the sum
    floatx4 o[DB], ol[split ? DB : 1];  // O^T: dims 16 db + 4 g16 .. +3; from P's high and low parts

    __device__ void start(int pos) {
        qpos = pos;
        m = kNone;
        l = 0.0f;
#pragma unroll
        for (int db = 0; db < DB; db++) {
            o[db] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (split) ol[db] = o[db];
        }
    }

    // q from the row at p (global memory or LDS), 16-byte aligned if vec
    __device__ void load(const typename PagedType<TYPE>::Io* p, bool vec, int g16, float qscale) {
        if constexpr (!split) {
            cs = qscale;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if (vec) q[ks] = *(const V8*)(p + 32 * ks + 8 * g16);
                else
#pragma unroll
                    for (int e = 0; e < 8; e++) q[ks][e] = p[32 * ks + 8 * g16 + e];
            }
        } else {
            float x[KS][8], mx = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float4 y = load4(p + 32 * ks + 8 * g16 + 4 * h, vec);
                    x[ks][4 * h] = y.x;
                    x[ks][4 * h + 1] = y.y;
                    x[ks][4 * h + 2] = y.z;
                    x[ks][4 * h + 3] = y.w;
                }
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[ks][e]));
            mx = max_x32(max_x16(mx));
            // 2^s with the largest element in [2^14, 2^15); 1 for zero and non-finite rows
            const int be = (int)((__float_as_uint(mx) >> 23) & 0xFFu);
            const int s = be == 0 || be == 255 ? 0 : min(141 - be, 126);
            const float up = power2(s);
            cs = qscale * power2(-s);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = x[ks][e] * up;
                    q[ks][e] = (_Float16)y;
                    ql[ks][e] = (_Float16)(y - (float)q[ks][e]);
                }
        }
    }
};

// One tile of KEYS keys from key0 on for RB row blocks. kl and vl: the tile in LDS. masked:
// some row of the wave ends inside the tile. LOW: P's low part of 16-bit rows as well.
template <int TYPE, int HD, int KEYS, int RB, bool LOW>
__device__ __forceinline__ void tile_step(RowBlock<TYPE, HD> (&rb)[RB], const char* kl, const char* vl, int key0, bool masked,
                                          const int (&koff)[Geo<HD>::KS], const int (&voff)[Geo<HD>::DB], int g16) {
    typedef Ops<TYPE> O;
    typedef typename O::V8 V8;
    typedef Geo<HD> G;
    constexpr int KB = KEYS / 16;
    floatx4 s[RB][KB];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int kb = 0; kb < KB; kb++) s[r][kb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++) {
        V8 kf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; kb++) kf[kb] = *(const V8*)(kl + koff[ks] + kb * G::BLKB);
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int kb = 0; kb < KB; kb++) s[r][kb] = O::mul(kf[kb], rb[r].q[ks], s[r][kb]);
        if constexpr (O::split) {
#pragma unroll
            for (int r = 0; r < RB; r++)
#pragma unroll
                for (int kb = 0; kb < KB; kb++) s[r][kb] = O::mul(kf[kb], rb[r].ql[ks], s[r][kb]);
        }
    }
    // The softmax goes ahead of the products of the SIMD's other wave, so that its own products are there sooner to
    // fill the matrix unit: 2048 tokens behind 6000 253 -> 242 us; with one row block nothing (16.9 and 17.5).
    if constexpr (RB > 1) __builtin_amdgcn_s_setprio(1);
    // keys key0 + 16 kb + 4 g16 + e of row c16
    constexpr bool low = O::split || LOW;
    V8 ph[RB][KB / 2], pl[low ? RB : 1][KB / 2];
#pragma unroll
    for (int r = 0; r < RB; r++) {
        RowBlock<TYPE, HD>& b = rb[r];
        if (masked) {
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (key0 + 16 * kb + 4 * g16 + e > b.qpos) s[r][kb][e] = -__builtin_huge_valf();
        }
        float mx = s[r][0][0];
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[r][kb][e]);
        mx = max_x32(max_x16(mx));
        if (__any((mx - b.m) * b.cs > kSlack)) {
            const float to = fmaxf(b.m, mx);
            const float corr = fast_exp2((b.m - to) * b.cs);
            b.m = to;
            b.l *= corr;
#pragma unroll
            for (int db = 0; db < G::DB; db++) {
                b.o[db] *= corr;
                if constexpr (O::split) b.ol[db] *= corr;
            }
        }
        // fp16's scale of P joins the exponent where half a step of fp16 hides its rounding
        const float mc = O::split ? b.m * b.cs : b.m * b.cs - (O::scale > 1.0f ? 11.0f : 0.0f);
        // k-step h: keys 4 g16 .. +3 of key block 2 h, then of block 2 h + 1
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float p = fast_exp2(fmaf(s[r][kb][e], b.cs, -mc));
                if constexpr (O::split) p *= O::scale;
                b.l += p;
                const auto hi = (typename PagedType<TYPE>::Page)p;
                ph[r][kb >> 1][4 * (kb & 1) + e] = hi;
                if constexpr (low)
                    pl[r][kb >> 1][4 * (kb & 1) + e] = (typename PagedType<TYPE>::Page)((p - (float)hi) * (O::split ? kLow : 1.0f));
            }
    }
    if constexpr (RB > 1) __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int h = 0; h < KB / 2; h++)
#pragma unroll
        for (int db = 0; db < G::DB; db++) {
            short4v part[2];
#pragma unroll
            for (int t = 0; t < 2; t++)
                part[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4v*)(vl + voff[db] + (2 * h + t) * G::BLKB));
            const short __attribute__((ext_vector_type(8))) both = {part[0][0], part[0][1], part[0][2], part[0][3],
                                                                    part[1][0], part[1][1], part[1][2], part[1][3]};
            const V8 vf = __builtin_bit_cast(V8, both);
#pragma unroll
            for (int r = 0; r < RB; r++) {
                rb[r].o[db] = O::mul(vf, ph[r][h], rb[r].o[db]);
                if constexpr (O::split) rb[r].ol[db] = O::mul(vf, pl[r][h], rb[r].ol[db]);
                else if constexpr (LOW) rb[r].o[db] = O::mul(vf, pl[r][h], rb[r].o[db]);
            }
        }
}

// Up to four rows again, packed rows r0 .. r0 + 3 of which those in `bad`, over their keys of tiles
// first, first + step, ... below end, in fp32 from q on. Row, maximum (log2 units) and sum of
// each go to res (rows of QS floats), m_out and l_out in the scale of the tiles' results. Lane = key
// for the scores, 64 keys at a time; lane = pair of dims for the sums over V. qs: room for
// four rows of QS floats.
template <int TYPE, int HD, int KEYS>
__device__ __forceinline__ void slow_rows(const PagedAttn& a, const Column& c, float* qs, int r0, unsigned bad, int first,
                                          int step, int end, int lane, float* res, float* m_out, float* l_out) {
    typedef typename PagedType<TYPE>::Io Io;
    typedef typename PagedType<TYPE>::Page Page;
    constexpr int QS = Geo<HD>::QS, NP = (HD / 2 + 63) / 64;
    constexpr int TPI = 64 / KEYS;  // tiles at a time
    int qp[4], qlast = -1;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int R = min(r0 + r, c.rows - 1);
        qp[r] = c.hist + R / a.g;
        qlast = max(qlast, qp[r]);
        const Io* p = (const Io*)a.q + row_offset<HD>(a, c, R, a.ldq);
        for (int e = lane; e < HD; e += 64) qs[r * QS + e] = (float)p[e] * a.qscale;
    }
    wave_sync();
    float m[4], l[4], acc[4][2 * NP];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        m[r] = kNone;
        l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NP; i++) acc[r][i] = 0.0f;
    }
#pragma unroll 1
    for (int kt = first; kt < end && kt * KEYS <= qlast; kt += TPI * step) {
        const int tile = kt + lane / KEYS * step, key = tile * KEYS + lane % KEYS;
        const bool in = tile < end && key <= qlast;
        const int at = in ? key : kt * KEYS;  // some key that exists
        const int pi = at >> a.shift;
        const int page = c.local ? c.local[pi] : a.pages[c.table + (c.list ? c.list[pi] : pi)];
        // within a layer's rows, which fit 31 bits
        const int krow = (int)((((unsigned)page * a.n_kv + c.kvh) << a.shift) + (at & ((1 << a.shift) - 1)));
        const u32x4* kr = (const u32x4*)(a.kp + (size_t)krow * Geo<HD>::ROWB);
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int ch = 0; ch < HD / 8; ch++) {
            const u32x4 u = kr[ch];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float* x = qs + r * QS + 8 * ch;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[r] = fmaf(x[2 * e], from_page<Page>((uint16_t)(u[e] & 0xFFFFu)), s[r]);
                    s[r] = fmaf(x[2 * e + 1], from_page<Page>((uint16_t)(u[e] >> 16)), s[r]);
                }
            }
        }
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const bool valid = in && key <= qp[r];
            const float sv = valid ? s[r] : -__builtin_huge_valf();
            const bool nan = __any(valid && !(s[r] == s[r]));
            const float mn = nan ? __builtin_nanf("") : fmaxf(m[r], group_max<64>(sv));
            const float corr = fast_exp2(m[r] - mn);
            p[r] = valid ? fast_exp2(sv - mn) * Ops<TYPE>::scale : 0.0f;
            l[r] = l[r] * corr + group_sum<64>(p[r]);
            m[r] = mn;
#pragma unroll
            for (int i = 0; i < 2 * NP; i++) acc[r][i] *= corr;
        }
        for (int j0 = 0; j0 < 64; j0 += 8) {
            uint32_t v[8][NP];
#pragma unroll
            for (int u = 0; u < 8; u++) {  // past the last key: the row of a key that exists, with weight 0 left out below
                const int vrow = __builtin_amdgcn_readlane(krow, j0 + u);
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const int d = 2 * (lane + 64 * i);
                    v[u][i] = d < HD ? *(const uint32_t*)(a.vp + (size_t)vrow * Geo<HD>::ROWB + 2 * d) : 0u;
                }
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int tj = kt + (j0 + u) / KEYS * step, kj = tj * KEYS + (j0 + u) % KEYS;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (tj >= end || kj > qp[r]) continue;
                    const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p[r]), j0 + u));
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        acc[r][2 * i] = fmaf(pj, from_page<Page>((uint16_t)(v[u][i] & 0xFFFFu)), acc[r][2 * i]);
                        acc[r][2 * i + 1] = fmaf(pj, from_page<Page>((uint16_t)(v[u][i] >> 16)), acc[r][2 * i + 1]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (!((bad >> r) & 1u)) continue;
#pragma unroll
        for (int i = 0; i < NP; i++)
            if (2 * (lane + 64 * i) < HD) *(float2*)(res + r * QS + 2 * (lane + 64 * i)) = float2{acc[r][2 * i], acc[r][2 * i + 1]};
        if (lane == 0) {
            m_out[r] = m[r];
            l_out[r] = l[r];
        }
    }
    wave_sync();
}

// A wave's row block to LDS: rows of QS floats at res, maximum (log2 units) and sum; rows that are
// not finite computed again over tiles first, first + step, ... below end.
template <int TYPE, int HD, int KEYS>
__device__ __forceinline__ void finish_rows(const PagedAttn& a, const Column& c, RowBlock<TYPE, HD>& b, int R0, int first,
                                            int step, int end, int lane, float* res, float* qs, float* m_out, float* l_out) {
    constexpr int DB = Geo<HD>::DB, QS = Geo<HD>::QS;
    const int c16 = lane & 15, g16 = lane >> 4;
    const float l = sum_x32(sum_x16(b.l));
    float chk = l * 0.0f;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (Ops<TYPE>::split) b.o[db][e] = fmaf(b.ol[db][e], 1.0f / kLow, b.o[db][e]);
            chk = fmaf(b.o[db][e], 0.0f, chk);
        }
    const bool sees = first < end && first * KEYS <= b.qpos;  // a key of these tiles
    const bool good = chk == 0.0f && (l > 0.0f || !sees);
    const unsigned long long lanes = __ballot(!good && R0 + c16 < c.rows);
    const unsigned bad = (unsigned)((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xFFFFu);
#pragma unroll
    for (int db = 0; db < DB; db++) *(floatx4*)(res + c16 * QS + 16 * db + 4 * g16) = b.o[db];
    if (g16 == 0) {
        m_out[c16] = b.m > kNone ? b.m * b.cs : kNone;
        l_out[c16] = l;
    }
    wave_sync();
    if (bad) {
#pragma unroll 1
        for (int r = 0; r < 16; r += 4)
            if ((bad >> r) & 15u)
                slow_rows<TYPE, HD, KEYS>(a, c, qs, R0 + r, bad >> r, first, step, end, lane, res + r * QS, m_out + r, l_out + r);
    }
}

// One output row's four elements: x / l, or 0 / 0 as the formula has it where every score is -inf.
template <int TYPE, int HD>
__device__ __forceinline__ void store_out(const PagedAttn& a, const Column& c, int R, int d, floatx4 x, float l) {
    typedef typename PagedType<TYPE>::Io Io;
    const float inv = 1.0f / l;
    Io* p = (Io*)a.out + row_offset<HD>(a, c, R, a.ldo) + d;
    store4(p, l == 0.0f ? float4{x[0] / l, x[1] / l, x[2] / l, x[3] / l} : float4{x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv},
           a.ovec);
}

// The parts of rows [r0, r0 + ROWS): part p at slot slot0 + p, rows of HD floats, then a
// maximum and a sum per row.
template <int HD, int ROWS>
struct Slots {
    static constexpr size_t FLOATS = (size_t)ROWS * (HD + 2);
};

// Partial results pass between workgroups on different dies, whose L2s are not coherent: stored
// and loaded past them (agent scope, relaxed), so that no cache has to be written back or emptied.
// (With a release and an acquire fence around plain accesses, which write back and empty an L2 per part,
// a token of 32 / 8 heads of 128 at 2048 keys took 18.1 us; so 10.9.)
__device__ __forceinline__ void part_store4(float* p, floatx4 x) {
    const auto u = __builtin_bit_cast(unsigned long long __attribute__((ext_vector_type(2))), x);
    __hip_atomic_store((unsigned long long*)p, (unsigned long long)u[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store((unsigned long long*)p + 1, (unsigned long long)u[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ floatx4 part_load4(const float* p) {
    unsigned long long __attribute__((ext_vector_type(2))) u;
    u[0] = __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    u[1] = __hip_atomic_load((const unsigned long long*)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return __builtin_bit_cast(floatx4, u);
}
// a row's maximum and sum
__device__ __forceinline__ void part_store2(float* p, float m, float l) {
    __hip_atomic_store((unsigned long long*)p, (unsigned long long)__float_as_uint(l) << 32 | __float_as_uint(m), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 part_load2(const float* p) {
    const unsigned long long u = __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((unsigned)u), __uint_as_float((unsigned)(u >> 32))};
}

// Joins the parts of `rows` rows in the order of the parts. lds: BYTES of the workgroup's LDS; the
// rows go in groups whose maxima and sums fit it. What costs time is the latency of the loads, so
// that 8 of a thread are on their way at once: of two elements of the rows where a group has more than the
// workgroup threads, else of one element's parts, which then several threads share. (16 took registers
// from the products: the wide kernel spilled.)
template <int TYPE, int HD, int ROWS, int BYTES>
__device__ __forceinline__ void join_parts(const PagedAttn& a, const Column& c, int slot0, int parts, int rows, char* lds) {
    constexpr int D4 = HD / 4, T = 2, U = 4;
    constexpr size_t F = Slots<HD, ROWS>::FLOATS;
    const float* base = a.part + (size_t)slot0 * F;
    const int tid = threadIdx.x, nt = blockDim.x;
    floatx4* s_a = (floatx4*)lds;                          // [threads]
    float* s_l = (float*)(lds + 16 * 256);                 // [ROWS] sums of all parts
    float2* s_w = (float2*)(lds + 16 * 256 + 4 * ROWS);    // [rows of a group][parts]: maximum (then weight) and sum
    const int fit = (BYTES - 16 * 256 - 4 * ROWS) / (8 * parts), step = min(rows, max(1, fit));
    for (int g0 = 0; g0 < rows; g0 += step) {
        const int n = min(step, rows - g0);
#pragma unroll 2
        for (int i = tid; i < n * parts; i += nt) {
            const int p = i / n, r = i - p * n;
            s_w[r * parts + p] = part_load2(base + p * F + ROWS * HD + 2 * (g0 + r));
        }
        __syncthreads();
        for (int r = tid; r < n; r += nt) {
            float2* w = s_w + r * parts;
            float M = kNone, L = 0.0f;
            bool nan = false;
            for (int p = 0; p < parts; p++) {
                nan |= !(w[p].x == w[p].x);
                M = fmaxf(M, w[p].x);
            }
            if (nan) M = __builtin_nanf("");
            for (int p = 0; p < parts; p++) {
                const float e = fast_exp2(w[p].x - M);
                L = fmaf(e, w[p].y, L);
                w[p].x = e;
            }
            s_l[r] = L;
        }
        __syncthreads();
        const int tasks = n * D4, share = max(1, min(parts, nt / tasks));
        if (share > 1) {
            const int j = tid / tasks, t = tid - j * tasks, r = t / D4, d = 4 * (t - r * D4);
            floatx4 A = {0.0f, 0.0f, 0.0f, 0.0f};
            if (j < share) {
                const float* src = base + (g0 + r) * HD + d;
#pragma unroll 1
                for (int p0 = j; p0 < parts; p0 += T * U * share) {
                    floatx4 x[T * U];  // past the last part: that one again, left out below
#pragma unroll
                    for (int u = 0; u < T * U; u++) x[u] = part_load4(src + min(p0 + u * share, parts - 1) * F);
#pragma unroll
                    for (int u = 0; u < T * U; u++)
                        if (p0 + u * share < parts) A += s_w[r * parts + p0 + u * share].x * x[u];
                }
            }
            s_a[tid] = A;
            __syncthreads();
            if (j == 0) {
                for (int u = 1; u < share; u++) A += s_a[tid + u * tasks];
                store_out<TYPE, HD>(a, c, c.r0 + g0 + r, d, A, s_l[r]);
            }
        } else {
#pragma unroll 1
            for (int i0 = tid; i0 < tasks; i0 += T * nt) {
                const int i1 = min(i0 + nt, tasks - 1);
                const float *s0 = base + g0 * HD + 4 * i0, *s1 = base + g0 * HD + 4 * i1;
                const float2 *w0 = s_w + i0 / D4 * parts, *w1 = s_w + i1 / D4 * parts;
                floatx4 A0 = {0.0f, 0.0f, 0.0f, 0.0f}, A1 = A0;
#pragma unroll 1
                for (int p0 = 0; p0 < parts; p0 += U) {
                    floatx4 x0[U], x1[U];  // past the last part: that one again, left out below
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const size_t at = min(p0 + u, parts - 1) * F;
                        x0[u] = part_load4(s0 + at);
                        x1[u] = part_load4(s1 + at);
                    }
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (p0 + u < parts) {
                            A0 += w0[p0 + u].x * x0[u];
                            A1 += w1[p0 + u].x * x1[u];
                        }
                }
                int r = i0 / D4;
                store_out<TYPE, HD>(a, c, c.r0 + g0 + r, 4 * (i0 - r * D4), A0, s_l[r]);
                r = i1 / D4;
                if (i0 + nt < tasks) store_out<TYPE, HD>(a, c, c.r0 + g0 + r, 4 * (i1 - r * D4), A1, s_l[r]);
            }
        }
        __syncthreads();
    }
}

// Parts of a column over chosen pages: as many as leave no workgroup idle, each with a tile per wave.
__host__ __device__ inline int chosen_parts(int wgs, int cols, int select, int shift) {
    if (cols <= 0) return 1;
    const long long keys = (long long)select << shift, piece = kNarrowKeys * kNarrowLeast;
    if (keys <= kNarrowKeys * kNarrowWhole) return 1;
    const long long most = (keys + piece - 1) / piece, room = wgs / cols;
    return (int)(room < 1 ? 1 : room < most ? room : most);
}

constexpr int narrow_waves(int hd) { return hd <= 128 ? 4 : 2; }

// Chosen pages of a column that one workgroup can hold besides its tiles.
constexpr int kFusedPages = 2048;

// ---- up to 16 rows: waves on different key tiles. CHOOSE: the workgroup makes the choice of its column's
// pages first, for single tokens: no second launch, and no column waits for the one with the most
// pages (32 tokens of 32 / 8 heads of 128, 32 of 125 to 886 pages each: 67.7 us in two launches, 57.9) ----
template <int TYPE, int HD, int KW, bool STREAM, bool CHOOSE>
__device__ __forceinline__ void narrow_body(const PagedAttn& a, const PagedChoose* ch) {
    typedef Geo<HD> G;
    typedef typename PagedType<TYPE>::Io Io;
    constexpr int KEYS = kNarrowKeys, KB = KEYS / 16;
    constexpr int LPW = 2 * KB * G::PPB;  // loads per tile
    constexpr int QB = HD * (int)sizeof(Io), QP = 16 * QB / 1024;  // bytes of a q row, 1 KB loads of 16 of them
    constexpr int D4 = HD / 4;
    __shared__ __attribute__((aligned(1024))) char lds[KW][2][2][KB * G::BLKB];  // [wave][buffer][K, V]
    __shared__ __attribute__((aligned(1024))) char sq[16 * QB];
    __shared__ float s_ml[KW][2][16];
    __shared__ int s_flag;
    __shared__ int s_page[CHOOSE ? kFusedPages : 1];

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g16 = lane >> 4;

    // lane offsets of a block's loads and of the operands in a tile
    unsigned goff[2][G::PPB];
#pragma unroll
    for (int i = 0; i < G::PPB; i++) {
        const int L = 64 * i + lane, r = L / G::CH, ch = L % G::CH;
        goff[0][i] = r * G::ROWB + 16 * (ch ^ G::xk(r));
        goff[1][i] = r * G::ROWB + 16 * (ch ^ G::xv(r));
    }
    int koff[G::KS], voff[G::DB];
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++) koff[ks] = c16 * G::ROWB + 16 * ((4 * ks + g16) ^ G::xk(c16));
    const int vr0 = 4 * g16 + (c16 >> 2);
#pragma unroll
    for (int db = 0; db < G::DB; db++)
        voff[db] = vr0 * G::ROWB + 16 * ((2 * db + ((c16 & 3) >> 1)) ^ G::xv(vr0)) + 8 * (c16 & 1);

    // the work: a run of the plan's items, or (chosen pages) columns of one token, KV head and 16
    // of its heads, each in as many parts as leave no workgroup idle
    const int n_blk = (a.g + 15) / 16;
    int it, it_end, it_step, rest, parts = 1, cols = 0;
    if (a.chosen) {
        cols = scalar_int(a.header, kHdTokens) * a.n_kv * n_blk;
        parts = chosen_parts(a.wgs, cols, a.select, a.shift);
        it = blockIdx.x;
        it_end = cols * parts;
        it_step = gridDim.x;
        rest = 0;
    } else {
        if ((int)blockIdx.x >= scalar_int(a.header, kHdRuns)) return;
        const int* run = a.runs + (size_t)blockIdx.x * (sizeof(PagedRun) / 4);
        it = 0;
        it_end = scalar_int(run, 0);
        rest = scalar_int(run, 1);
        it_step = 1;
    }
    for (; it < it_end; it += it_step) {
        Column c;
        int t0, t1, slot0, part, counter;
        if (a.chosen) {
            const int col = it / parts;
            part = it - col * parts;
            const int blk = col % n_blk, tk = col / n_blk, tok = tk / a.n_kv;
            const int pos = scalar_int(a.tokens, 4 * tok + 1);
            const int seen = min(a.select, (pos >> a.shift) + 1);  // pages, the last of them the token's own
            c.kend = ((seen - 1) << a.shift) + (pos & ((1 << a.shift) - 1)) + 1;
            c.row0 = tok;
            c.rows = a.g;
            c.hist = c.kend - 1;
            c.table = scalar_int(a.tokens, 4 * tok);
            c.kvh = tk - tok * a.n_kv;
            c.r0 = 16 * blk;
            c.list = CHOOSE ? nullptr : a.chosen + (size_t)tk * a.select;
            c.local = nullptr;
            if constexpr (CHOOSE) {
                __shared__ ListScratch scratch;
                const int n = (pos >> a.shift) + 1;
                if (n > a.select) {
                    uint32_t* room = (uint32_t*)&lds[0][0][0][0];
                    score_pages<TYPE, HD, (HD <= 128 ? 8 : 4)>(*ch, room, tok, 1, c.kvh, c.table, ch->first, n - ch->last, w, KW);
                    __syncthreads();
                    const Keys keys = {room, ch->first, n - ch->last, n};
                    if (n > kWaveKeys) choose_by_block(keys, a.select, scratch, w, KW, s_page);
                    else if (w == 0) {
                        if (n <= 256) choose_by_wave<4>(keys, a.select, lane, s_page);
                        else if (n <= 512) choose_by_wave<8>(keys, a.select, lane, s_page);
                        else if (n <= 768) choose_by_wave<12>(keys, a.select, lane, s_page);
                        else choose_by_wave<16>(keys, a.select, lane, s_page);
                    }
                } else {
                    for (int i = tid; i < n; i += 64 * KW) s_page[i] = i;
                }
                __syncthreads();
                int* out = ch->chosen + (size_t)tk * a.select;
                for (int i = tid; i < a.select; i += 64 * KW) {
                    const int p = i < seen ? s_page[i] : -1;
                    if (part == 0 && blk == 0) out[i] = p;
                    if (p >= 0) s_page[i] = a.pages[c.table + p];
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no store among the counted loads
                __syncthreads();
                c.local = s_page;
            }
            const int tiles = (c.kend + KEYS - 1) / KEYS;
            t0 = (int)((long long)tiles * part / parts);
            t1 = (int)((long long)tiles * (part + 1) / parts);
            slot0 = col * parts;
            counter = col;
        } else {
            const int* p = it == 0 ? a.runs + (size_t)blockIdx.x * (sizeof(PagedRun) / 4) + 4
                                   : a.items + (size_t)(rest + it - 1) * (sizeof(PagedItem) / 4);
            c.row0 = scalar_int(p, 0);
            c.rows = scalar_int(p, 1);
            c.hist = scalar_int(p, 2);
            c.table = scalar_int(p, 3);
            c.kvh = scalar_int(p, 4);
            c.r0 = scalar_int(p, 5);
            t0 = scalar_int(p, 6);
            t1 = scalar_int(p, 7);
            slot0 = scalar_int(p, 8);
            part = scalar_int(p, 9);
            parts = scalar_int(p, 10);
            counter = scalar_int(p, 11);
            c.kend = c.hist + (c.rows - 1) / a.g + 1;
            c.list = nullptr;
            c.local = nullptr;
        }
        const int nrow = min(16, c.rows - c.r0);
        const int tile0 = t0 + w;  // this wave's tiles: tile0, tile0 + KW, ...

        int page[KB];  // of the tile that is loaded next
        auto look = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < KB; b++) page[b] = page_at(a, c, min(kt * KEYS + 16 * b, c.kend - 1) >> a.shift);
        };
        auto issue = [&](int kt, int buf) __attribute__((always_inline)) {
            if (kt >= t1) return;
#pragma unroll
            for (int b = 0; b < KB; b++) {
                const int pos = min(kt * KEYS + 16 * b, (c.kend - 1) & ~15);  // a block past the last one: that one again
                const size_t at = block_offset<HD>(a, c, page[b], pos);
                const int last = c.kend - 1 - pos;  // rows past the last key repeat it (and are masked)
#pragma unroll
                for (int o = 0; o < 2; o++) {
                    const char* src = (o ? a.vp : a.kp) + at;
#pragma unroll
                    for (int i = 0; i < G::PPB; i++) {
                        unsigned off = goff[o][i];
                        if (last < 15) {
                            const int L = 64 * i + lane, r = L / G::CH;
                            off = min(r, last) * G::ROWB + 16 * ((L % G::CH) ^ (o ? G::xv(r) : G::xk(r)));
                        }
                        if constexpr (STREAM) lds_dma_b128_nt(src, off, lds_addr(&lds[w][buf][o][b * G::BLKB + 1024 * i]));
                        else lds_dma_b128(src, off, lds_addr(&lds[w][buf][o][b * G::BLKB + 1024 * i]));
                    }
                }
            }
            if (kt + KW < t1) look(kt + KW);
        };
        if (tile0 < t1) look(tile0);
        // q ahead of the tiles, so that the wave can wait for it alone
        const Io* q = (const Io*)a.q;
        if (a.qvec) {
            for (int i = w; i < QP; i += KW) {
                const int L = 64 * i + lane, r = L / (QB / 16);
                const char* p = (const char*)(q + row_offset<HD>(a, c, c.r0 + min(r, nrow - 1), a.ldq)) + 16 * (L % (QB / 16));
                lds_dma_b128_at(p, lds_addr(sq + 1024 * i));
            }
        } else {
            for (int i = tid; i < 16 * HD; i += 64 * KW) {
                const int r = i / HD;
                ((Io*)sq)[i] = q[row_offset<HD>(a, c, c.r0 + min(r, nrow - 1), a.ldq) + i - r * HD];
            }
        }
        issue(tile0, 0);
        issue(tile0 + KW, 1);
        const int mine = tile0 >= t1 ? 0 : tile0 + KW >= t1 ? 1 : 2;
        if (mine == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LPW < 63 ? 2 * LPW : 63) : "memory");
        else if (mine == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPW < 63 ? LPW : 63) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        RowBlock<TYPE, HD> rb[1];
        rb[0].load((const Io*)sq + c16 * HD, true, g16, a.qscale);
        rb[0].start(c.hist + min(c.r0 + c16, c.rows - 1) / a.g);
        const int qmin = c.hist + c.r0 / a.g;

        int buf = 0;
        for (int kt = tile0; kt < t1; kt += KW) {
            if (kt + KW < t1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPW < 63 ? LPW : 63) : "memory");  // the next tile's stay in flight
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            tile_step<TYPE, HD, KEYS, 1, KW == narrow_waves(HD)>(rb, lds[w][buf][0], lds[w][buf][1], kt * KEYS,
                                                                 kt * KEYS + KEYS - 1 > qmin, koff, voff, g16);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the buffer has been read
            issue(kt + 2 * KW, buf);
            buf ^= 1;
        }

        // the waves' results to their own tile buffers, then together
        float* res = (float*)&lds[w][0][0][0];
        finish_rows<TYPE, HD, KEYS>(a, c, rb[0], c.r0, tile0, KW, t1, lane, res, res + 16 * G::QS, s_ml[w][0], s_ml[w][1]);
        __syncthreads();
        float* slot = a.part + (size_t)(slot0 + part) * Slots<HD, 16>::FLOATS;
        for (int i = tid; i < nrow * D4; i += 64 * KW) {
            const int r = i / D4, d = 4 * (i - r * D4);
            float M = kNone, L = 0.0f;
            bool nan = false;
            floatx4 A = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KW; k++) {
                const float m = s_ml[k][0][r];
                nan |= !(m == m);
                M = fmaxf(M, m);
            }
            if (nan) M = __builtin_nanf("");
#pragma unroll
            for (int k = 0; k < KW; k++) {
                const float e = fast_exp2(s_ml[k][0][r] - M);
                L = fmaf(e, s_ml[k][1][r], L);
                A += e * *(const floatx4*)((const float*)&lds[k][0][0][0] + r * G::QS + d);
            }
            if (parts > 1) {
                part_store4(slot + r * HD + d, A);
                if (d == 0) part_store2(slot + 16 * HD + 2 * r, M, L);
            } else {
                store_out<TYPE, HD>(a, c, c.r0 + r, d, A, L);
            }
        }
        if (parts > 1 && last_of(a.counters + counter, parts, &s_flag)) 
            join_parts<TYPE, HD, 16, (int)sizeof lds>(a, c, slot0, parts, nrow, &lds[0][0][0][0]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no store among the next item's counted loads
        __syncthreads();  // LDS is free again
    }
}

template <int TYPE, int HD, int KW, bool STREAM>
__global__ __launch_bounds__(64 * KW, KW == 4 && HD == 64 ? 2 : 1) void paged_narrow_kernel(const PagedAttn a) {
    narrow_body<TYPE, HD, KW, STREAM, false>(a, nullptr);
}

template <int TYPE, int HD, int KW, bool STREAM>
__global__ __launch_bounds__(64 * KW, KW == 4 && HD == 64 ? 2 : 1) void paged_sparse_kernel(const PagedAttn a, const PagedChoose ch) {
    narrow_body<TYPE, HD, KW, STREAM, true>(a, &ch);
}

// blocks of 16 rows per wave: two share each operand read where the registers hold them; one for batches
// that would leave CUs idle
constexpr int wide_blocks(int type, int hd) { return type != PQA_PAGED_F32 && hd <= 128 ? 2 : 1; }
template <int HD>
constexpr int wide_keys() { return HD > 192 ? 32 : 64; }

// ---- more rows: 4 waves share each key tile, RB blocks of 16 rows each ----
template <int TYPE, int HD, int RB>
__global__ __launch_bounds__(256, HD == 64 ? 3 : HD <= 128 ? 2 : 1) void paged_wide_kernel(const PagedAttn a) {
    typedef Geo<HD> G;
    typedef typename PagedType<TYPE>::Io Io;
    constexpr int KEYS = wide_keys<HD>(), KB = KEYS / 16, ROWS = 64 * RB;
    constexpr int D4 = HD / 4;
    constexpr int TILE = KB * G::BLKB;
    constexpr int WAVE = 20 * G::QS * 4;  // a wave's result and its slow rows' q
    constexpr int BYTES = 4 * TILE > 4 * WAVE ? 4 * TILE : 4 * WAVE;
    __shared__ __attribute__((aligned(1024))) char lds[BYTES];  // [buffer][K, V][TILE]
    __shared__ float s_ml[4][2][16];
    __shared__ int s_flag;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g16 = lane >> 4;
    // the wave's share of a tile's loads: block lb of 16 keys, operands lo0 .. lo1
    constexpr int OPS = KB == 4 ? 2 : 1;
    const int lb = w & (KB - 1), lo0 = KB == 4 ? 0 : w >> 1;
    int koff[G::KS], voff[G::DB];
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++) koff[ks] = c16 * G::ROWB + 16 * ((4 * ks + g16) ^ G::xk(c16));
    const int vr0 = 4 * g16 + (c16 >> 2);
#pragma unroll
    for (int db = 0; db < G::DB; db++)
        voff[db] = vr0 * G::ROWB + 16 * ((2 * db + ((c16 & 3) >> 1)) ^ G::xv(vr0)) + 8 * (c16 & 1);
    unsigned goff[OPS][G::PPB];
#pragma unroll
    for (int o = 0; o < OPS; o++)
#pragma unroll
        for (int i = 0; i < G::PPB; i++) {
            const int L = 64 * i + lane, r = L / G::CH;
            goff[o][i] = r * G::ROWB + 16 * ((L % G::CH) ^ (lo0 + o ? G::xv(r) : G::xk(r)));
        }

    const int n_items = scalar_int(a.header, RB == wide_blocks(TYPE, HD) ? kHdWide : kHdSmall);
    for (int it = blockIdx.x; it < n_items; it += gridDim.x) {
        const int* p = a.items + (size_t)it * (sizeof(PagedItem) / 4);
        Column c;
        c.row0 = scalar_int(p, 0);
        c.rows = scalar_int(p, 1);
        c.hist = scalar_int(p, 2);
        c.table = scalar_int(p, 3);
        c.kvh = scalar_int(p, 4);
        c.r0 = scalar_int(p, 5);
        const int t0 = scalar_int(p, 6), t1 = scalar_int(p, 7), slot0 = scalar_int(p, 8), part = scalar_int(p, 9),
                  parts = scalar_int(p, 10), counter = scalar_int(p, 11);
        c.kend = c.hist + (c.rows - 1) / a.g + 1;
        c.list = nullptr;
        c.local = nullptr;

        int page;  // of the wave's block in the tile that is loaded next
        auto look = [&](int kt) __attribute__((always_inline)) {
            page = page_at(a, c, min(kt * KEYS + 16 * lb, c.kend - 1) >> a.shift);
        };
        auto issue = [&](int kt, int buf) __attribute__((always_inline)) {
            if (kt >= t1) return;
            const int pos = min(kt * KEYS + 16 * lb, (c.kend - 1) & ~15);
            const size_t at = block_offset<HD>(a, c, page, pos);
            const int last = c.kend - 1 - pos;
#pragma unroll
            for (int o = 0; o < OPS; o++) {
                const char* src = (lo0 + o ? a.vp : a.kp) + at;
#pragma unroll
                for (int i = 0; i < G::PPB; i++) {
                    unsigned off = goff[o][i];
                    if (last < 15) {
                        const int L = 64 * i + lane, r = L / G::CH;
                        off = min(r, last) * G::ROWB + 16 * ((L % G::CH) ^ (lo0 + o ? G::xv(r) : G::xk(r)));
                    }
                    lds_dma_b128(src, off, lds_addr(lds + (2 * buf + lo0 + o) * TILE + lb * G::BLKB + 1024 * i));
                }
            }
            if (kt + 1 < t1) look(kt + 1);
        };
        const int R0 = c.r0 + 16 * RB * w;  // the wave's rows
        RowBlock<TYPE, HD> rb[RB];
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const int R = min(R0 + 16 * r + c16, c.rows - 1);
            rb[r].load((const Io*)a.q + row_offset<HD>(a, c, R, a.ldq), a.qvec, g16, a.qscale);
            rb[r].start(c.hist + R / a.g);
        }
        const int qmin = c.hist + min(R0, c.rows - 1) / a.g;
        const int qmax = R0 < c.rows ? c.hist + min(R0 + 16 * RB - 1, c.rows - 1) / a.g : -1;
        look(t0);
        issue(t0, 0);
        int buf = 0;
        for (int kt = t0; kt < t1; kt++) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the tile
            __syncthreads();                                   // everyone's; the other buffer is free
            issue(kt + 1, buf ^ 1);
            if (kt * KEYS <= qmax)
                tile_step<TYPE, HD, KEYS, RB, false>(rb, lds + 2 * buf * TILE, lds + (2 * buf + 1) * TILE, kt * KEYS,
                                              kt * KEYS + KEYS - 1 > qmin, koff, voff, g16);
            buf ^= 1;
        }
        __syncthreads();  // the tiles have been read
        float* res = (float*)(lds + w * WAVE);
        float* slot = a.part + (size_t)(slot0 + part) * Slots<HD, ROWS>::FLOATS;
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const int first = R0 + 16 * r, n = min(16, c.rows - first);
            if (n <= 0) break;
            finish_rows<TYPE, HD, KEYS>(a, c, rb[r], first, t0, 1, t1, lane, res, res + 16 * G::QS, s_ml[w][0], s_ml[w][1]);
            for (int i = lane; i < n * D4; i += 64) {
                const int j = i / D4, d = 4 * (i - j * D4), at = 16 * (RB * w + r) + j;
                const floatx4 x = *(const floatx4*)(res + j * G::QS + d);
                if (parts > 1) {
                    part_store4(slot + at * HD + d, x);
                    if (d == 0) part_store2(slot + ROWS * HD + 2 * at, s_ml[w][0][j], s_ml[w][1][j]);
                } else {
                    store_out<TYPE, HD>(a, c, first + j, d, x, s_ml[w][1][j]);
                }
            }
            wave_sync();
        }
        if (parts > 1 && last_of(a.counters + counter, parts, &s_flag))
            join_parts<TYPE, HD, ROWS, BYTES>(a, c, slot0, parts, min(ROWS, c.rows - c.r0), lds);
        __syncthreads();  // LDS is free again
    }
}

// Which kernels a call launches, on how many workgroups (0: not at all).
struct Launch {
    int narrow_grid, wide_grid;
    const PagedChoose* choose;  // the narrow kernel makes the choice of its pages, or null
    bool stream, small, captured;
};

template <int TYPE, int HD>
hipError_t launch_kernels(const PagedAttn& a, const PagedAttn& wide, const Launch& l, hipStream_t s) {
    if (l.narrow_grid) {
        constexpr int KW = narrow_waves(HD);
        const dim3 grid((unsigned)l.narrow_grid);
        if (l.choose) {
            if (l.stream) hipLaunchKernelGGL((paged_sparse_kernel<TYPE, HD, KW, true>), grid, dim3(64 * KW), 0, s, a, *l.choose);
            else hipLaunchKernelGGL((paged_sparse_kernel<TYPE, HD, KW, false>), grid, dim3(64 * KW), 0, s, a, *l.choose);
        } else if (l.stream) hipLaunchKernelGGL((paged_narrow_kernel<TYPE, HD, KW, true>), grid, dim3(64 * KW), 0, s, a);
        else if (a.crowd) hipLaunchKernelGGL((paged_narrow_kernel<TYPE, HD, 2, false>), grid, dim3(128), 0, s, a);
        else hipLaunchKernelGGL((paged_narrow_kernel<TYPE, HD, KW, false>), grid, dim3(64 * KW), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    // a captured call launches both tiles; the one that the batch's items are not made for finds none
    constexpr int RB = wide_blocks(TYPE, HD);
    if (l.wide_grid && (l.captured || !l.small)) {
        hipLaunchKernelGGL((paged_wide_kernel<TYPE, HD, RB>), dim3((unsigned)l.wide_grid), dim3(256), 0, s, wide);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if constexpr (RB > 1)
        if (l.wide_grid && (l.captured || l.small)) {
            hipLaunchKernelGGL((paged_wide_kernel<TYPE, HD, 1>), dim3((unsigned)l.wide_grid), dim3(256), 0, s, wide);
            return hipGetLastError();
        }
    return hipSuccess;
}

template <int TYPE>
hipError_t launch_type(int hd, const PagedAttn& a, const PagedAttn& wide, const Launch& l, hipStream_t s) {
    switch (hd) {
#define PQA_PG(H) case H: return launch_kernels<TYPE, H>(a, wide, l, s);
        PQA_PG(64) PQA_PG(96) PQA_PG(128) PQA_PG(160) PQA_PG(192) PQA_PG(256)
#undef PQA_PG
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_any(const pqa_batch* b, const PagedAttn& a, const PagedAttn& wide, const Launch& l, hipStream_t s) {
    switch (b->p->type) {
        case PQA_PAGED_F32: return launch_type<PQA_PAGED_F32>(b->p->head_dim, a, wide, l, s);
        case PQA_PAGED_F16: return launch_type<PQA_PAGED_F16>(b->p->head_dim, a, wide, l, s);
        default: return launch_type<PQA_PAGED_BF16>(b->p->head_dim, a, wide, l, s);
    }
}

PagedAttn arguments(const pqa_batch* b, int layer, const PagedRows& q, void* out, long long ldo) {
    const pqa_paged* p = b->p;
    const size_t io = (size_t)paged_io_bytes(p->type);
    PagedAttn a{};
    a.q = q.p;
    a.out = out;
    a.ldq = q.ld;
    a.ldo = ldo;
    a.kp = p->k + (size_t)layer * p->layer_bytes;
    a.vp = p->v + (size_t)layer * p->layer_bytes;
    a.pages = b->pages;
    a.items = (const int*)b->rest;
    a.runs = (const int*)b->runs;
    a.header = b->header;
    a.part = b->part_narrow;
    a.counters = b->counters;
    a.tokens = (const int*)b->tokens;
    a.wgs = b->shape.narrow_wgs;
    a.g = p->group;
    a.n_kv = p->n_kv;
    a.shift = p->page_shift;
    a.qvec = ((uintptr_t)q.p & 15) == 0 && q.ld * io % 16 == 0;
    a.ovec = ((uintptr_t)out & (4 * io - 1)) == 0 && ldo % 4 == 0;
    a.qscale = 1.4426950408889634f / sqrtf((float)p->head_dim);
    return a;
}

}  // namespace

int paged_wide_rows(int type, int hd) { return 64 * wide_blocks(type, hd); }
int paged_least_rows() { return 64; }
int paged_wide_keys(int hd) { return hd > 192 ? 32 : 64; }
int paged_narrow_wgs(int hd, int cu_count) { return hd == 64 ? 2 * cu_count : cu_count; }
int paged_wide_wgs(int hd, int cu_count) { return hd == 64 ? 3 * cu_count : hd <= 128 ? 2 * cu_count : cu_count; }

hipError_t launch_paged_attend(const pqa_batch* b, int layer, const PagedRows& q, void* out, long long ldo, bool captured,
                               hipStream_t s) {
    const PagedAttn a = arguments(b, layer, q, out, ldo);
    PagedAttn wide = a;
    wide.items = (const int*)b->wide;
    wide.part = b->part_wide;
    wide.counters = b->counters + b->shape.narrow_wgs;
    // A captured call may be replayed with what the batch holds then: both kernels, on grids that
    // any content fits
    const int n = captured ? b->shape.narrow_wgs : (int)b->plan.runs.size();
    const int w = captured ? b->shape.wide_wgs : (int)b->plan.wide.size();
    return launch_any(b, a, wide, {n, w, nullptr, b->plan.stream, b->plan.wide_rows < b->shape.wide_rows, captured}, s);
}

hipError_t launch_paged_sparse(const pqa_batch* b, int layer, const PagedRows& q, int select, int first, int last, int* chosen,
                               void* out, long long ldo, bool captured, hipStream_t s) {
    const pqa_paged* p = b->p;
    PagedAttn a = arguments(b, layer, q, out, ldo);
    a.chosen = chosen;
    a.select = select;
    PagedChoose ch = choose_arguments(b, layer, q, select, first, last, chosen, captured);
    const long long cols = (long long)b->plan.n_tok * p->n_kv * ((p->group + 15) / 16);
    const long long grid = captured ? b->shape.narrow_wgs : cols * chosen_parts(a.wgs, (int)cols, select, a.shift);
    // tokens of one sequence share the loads of a choice, and long columns its work: a launch of its own for these
    const bool tokens = captured ? b->shape.max_tokens <= b->shape.max_seqs : ch.single;
    // (and where 16 heads are not all: a workgroup of the others may write their rows, which the choice reads,
    // if out is q)
    const bool fused = tokens && ch.parts == 1 && p->group <= 16 && select <= kFusedPages &&
                       4 * ch.stride <= narrow_waves(p->head_dim) * 2 * kNarrowKeys * 4 * p->head_dim;
    if (!fused) {
        const hipError_t e = launch_paged_choose(b, ch, captured, s);
        if (e != hipSuccess) return e;
    }
    a.crowd = !fused && cols >= 2 * a.wgs;
    // chosen pages of single tokens are read once, those of a chunk's tokens by many of them
    const bool stream = ch.single && cols * ((long long)select << a.shift) * 4 * p->head_dim > kStreamBytes;
    return launch_any(b, a, a, {(int)std::min<long long>(grid, 1 << 30), 0, fused ? &ch : nullptr, stream, false, captured}, s);
}

}  // namespace pqa
