// The batch of a paged call: its checks, its tables and how its attention work is cut
// into pieces for the workgroups. Host code without HIP, so that the CPU tests can build
// it.
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

namespace pqa {

// Rows of one workgroup tile. A row is one query head of one new token; the rows of a
// sequence and KV head are packed token by token, so that heads that share a KV head share
// its loads. Up to kNarrowRows rows a sequence's work is bound by reading K and V: one block
// of 16 rows, whose waves take the key tiles in turn. More rows go to tiles of
// paged_wide_rows, whose waves share each key tile.
constexpr int kNarrowRows = 16;
constexpr int kNarrowKeys = 32;  // keys per tile of a wave

// One piece of work: rows [r0, r0 + tile rows) of a sequence and KV head against the key
// tiles [t0, t1). With parts > 1 the keys of these rows are cut and each piece leaves
// partial results at its slot; the last of the parts to finish joins slots slot0, slot0 + 1, ...
struct PagedItem {
    int32_t row0;   // first token row of the sequence
    int32_t rows;   // packed rows of the sequence (new tokens x heads per KV head)
    int32_t hist;   // position of its first new token
    int32_t table;  // its first entry in the page list
    int32_t kvh, r0, t0, t1;
    int32_t slot0, part, parts, counter;
};

struct PagedSeq {
    int32_t row0, n_new, len, table;
};

struct PagedToken {  // a token row: its sequence's page list, its position, its number among the sequence's new ones, and
    int32_t table, pos, nth, left;  // how many of these there are from it on
};

struct PagedRun {  // a narrow workgroup's items: the first, and count - 1 more from `rest` on
    int32_t count, rest, unused[2];
    PagedItem first;
};

struct PagedTouched {  // a page that receives rows: its id and the rows in use afterwards
    int32_t page, used;
};

// What the handle fixes: sizes and how much runs at once.
struct PagedShape {
    int n_pages, page_size, group, n_kv, max_pos;  // max_pos: positions that the rotation's tables hold; 0: no rotation
    int narrow_wgs;                                // workgroups of the narrow kernel that run at once
    int wide_wgs, wide_rows, wide_keys;            // the same for the wide one, and its largest tile
    int least_rows;                                // rows of its smaller tile, or wide_rows
    int key_bytes;                                 // K and V of one position and KV head
    int max_seqs, max_tokens, max_seq_pages;       // what the batch holds; pages of one sequence
};

struct PagedPlan {
    int n_tok = 0;
    std::vector<PagedSeq> seqs;
    std::vector<PagedToken> tokens;
    std::vector<int32_t> pages;
    std::vector<PagedTouched> touched;
    std::vector<PagedRun> runs;  // of the narrow workgroups that have work
    std::vector<PagedItem> rest, wide;
    int wide_rows = 0;    // of the wide items' tile
    bool stream = false;  // the narrow items' K and V pass through the caches once
};

enum class PagedFault { none, argument, range };

// Slots of partial results that a plan may use. A narrow workgroup's items are a run of the
// columns, so only its first and last can be cut; a wide plan keeps to its own bound.
inline int paged_narrow_slots(const PagedShape& s) { return 2 * s.narrow_wgs; }
inline int paged_wide_slots(const PagedShape& s) { return 2 * s.wide_wgs; }

// Fills the sequences, the page list and the touched pages, or says what is wrong.
inline PagedFault paged_check(const PagedShape& s, int n_seqs, const int* n_new, const int* len, const int* pages,
                              int stride, PagedPlan* plan, std::string* why) {
    char text[200];
    auto fail = [&](PagedFault f) {
        *why = text;
        return f;
    };
    plan->seqs.clear();
    plan->tokens.clear();
    plan->pages.clear();
    plan->touched.clear();
    if (n_seqs < 0 || n_seqs > s.max_seqs) {
        std::snprintf(text, sizeof text, "%d sequences, the batch holds 0 to %d", n_seqs, s.max_seqs);
        return fail(PagedFault::argument);
    }
    if (n_seqs > 0 && (!n_new || !len || !pages)) {
        std::snprintf(text, sizeof text, "NULL array");
        return fail(PagedFault::argument);
    }
    long long tokens = 0, entries = 0;
    for (int i = 0; i < n_seqs; i++) {
        if (n_new[i] < 0 || len[i] < n_new[i]) {
            std::snprintf(text, sizeof text, "sequence %d: %d new tokens of %d in all", i, n_new[i], len[i]);
            return fail(PagedFault::argument);
        }
        if (s.max_pos > 0 && len[i] > s.max_pos) {
            std::snprintf(text, sizeof text, "sequence %d: length %d, the rotation's tables end at %d", i, len[i], s.max_pos);
            return fail(PagedFault::range);
        }
        const int used = (int)(((long long)len[i] + s.page_size - 1) / s.page_size);
        if (used > stride || used > s.max_seq_pages) {
            std::snprintf(text, sizeof text, "sequence %d: length %d takes %d pages, its list holds %d and the batch %d", i, len[i],
                          used, stride, s.max_seq_pages);
            return fail(PagedFault::range);
        }
        tokens += n_new[i];
        entries += used;
    }
    if (tokens > s.max_tokens) {
        std::snprintf(text, sizeof text, "%lld new tokens, the batch holds %d", tokens, s.max_tokens);
        return fail(PagedFault::range);
    }
    plan->n_tok = (int)tokens;
    plan->seqs.reserve(n_seqs);
    plan->tokens.reserve((size_t)tokens);
    plan->pages.reserve((size_t)entries);
    // a page that receives rows belongs to one sequence alone: 1 listed, 2 listed and written
    std::vector<char> mark((size_t)s.n_pages, 0);
    for (int pass = 0; pass < 2; pass++)
        for (int i = 0; i < n_seqs; i++) {
            const int used = (int)(((long long)len[i] + s.page_size - 1) / s.page_size);
            const int first = n_new[i] ? (len[i] - n_new[i]) / s.page_size : used;  // pages from here on receive rows
            for (int j = 0; j < used; j++) {
                const int p = pages[(size_t)i * stride + j];
                const bool written = j >= first;
                if (pass == 0) {
                    if (p < 0 || p >= s.n_pages) {
                        std::snprintf(text, sizeof text, "sequence %d: page %d at place %d, there are %d", i, p, j, s.n_pages);
                        return fail(PagedFault::argument);
                    }
                    if (written) {
                        if (mark[p]) {
                            std::snprintf(text, sizeof text, "page %d receives rows of sequence %d and is listed twice", p, i);
                            return fail(PagedFault::argument);
                        }
                        mark[p] = 2;
                    }
                } else if (!written && mark[p] == 2) {
                    std::snprintf(text, sizeof text, "page %d of sequence %d receives rows of another place of the batch", p, i);
                    return fail(PagedFault::argument);
                }
            }
        }
    int row = 0;
    for (int i = 0; i < n_seqs; i++) {
        const int used = (int)(((long long)len[i] + s.page_size - 1) / s.page_size);
        plan->seqs.push_back({row, n_new[i], len[i], (int)plan->pages.size()});
        for (int j = 0; j < n_new[i]; j++) plan->tokens.push_back({(int)plan->pages.size(), len[i] - n_new[i] + j, j, n_new[i] - j});
        plan->pages.insert(plan->pages.end(), pages + (size_t)i * stride, pages + (size_t)i * stride + used);
        if (n_new[i])
            for (int j = (len[i] - n_new[i]) / s.page_size; j < used; j++)
                plan->touched.push_back({pages[(size_t)i * stride + j], std::min(s.page_size, len[i] - j * s.page_size)});
        row += n_new[i];
    }
    return PagedFault::none;
}

// Which kernel takes a sequence of few rows. Beside chunks the wide one does, as long as its keys are
// few: one launch, and the chunks' workgroups fill the gaps (3 chunks of 150 to 500 tokens beside 9
// single ones behind 10 to 4000, fp32, 32 / 4 heads of 64: 30.0 us in two launches, 16.9 in one). From
// kWideBytes on the narrow one's rate is worth its launch (a chunk of 100 beside 32 tokens behind 3000,
// bf16, 32 / 8 heads of 128, 393 MB: 83 us in one, 76 in two; behind 8000 188 and 170).
constexpr long long kWideBytes = 96LL << 20;
// K and V of this many bytes and more go past the L2s (32 MB in all), which then keep what the call
// reads again: 131072 keys of 8 heads of 128 (537 MB) 101 -> 90 us, 48 tokens behind 345k positions 205 ->
// 183. Below, a caller that comes back to the same layer soon finds them there: 700 keys of 2 heads of
// 64 8.4 us, past the caches 9.3.
constexpr long long kStreamBytes = 48LL << 20;

// The narrow items: the key tiles of all (sequence, KV head) columns laid end to end and cut
// into a run per workgroup. A column costs its tiles and kNarrowOverhead more (q, the joining
// of the waves, the write), a run has at least kNarrowLeast tiles (one per wave), and a cut
// leaves at least that much on both sides. Where no column is longer than kNarrowWhole tiles none is
// cut below its length: joining parts costs what those tiles do.
constexpr int kNarrowOverhead = 8;
constexpr int kNarrowLeast = 4;
constexpr int kNarrowWhole = 24;

// The wide items: blocks of rows, longest first, cut along the keys into parts of about an even share of all
// blocks' tiles and at least kWideLeast keys. Blocks are of wide_rows unless these are fewer than the
// workgroups that run at once, then of least_rows (bf16, 32 / 8 heads of 128: 512 tokens 21.3 us in blocks of 128, 13.2
// of 64; 64 behind 3000 37.9 and 24.5; 2048 62.7 and 61.0; 6 x 1000 behind 0 to 2500 224 and 258).
constexpr int kWideLeast = 512;

inline void paged_items(const PagedShape& s, PagedPlan* plan) {
    plan->runs.clear();
    plan->rest.clear();
    plan->wide.clear();
    std::vector<PagedItem> items;
    std::vector<int> first;  // of each workgroup
    long long cost = 0, bytes = 0;
    int longest = 0;
    bool chunks = false;
    for (const PagedSeq& q : plan->seqs) {
        if (!q.n_new) continue;
        if ((long long)q.n_new * s.group > kNarrowRows) {
            chunks = true;
            continue;
        }
        const int tiles = (q.len + kNarrowKeys - 1) / kNarrowKeys;
        longest = std::max(longest, tiles);
        cost += (long long)s.n_kv * (tiles + kNarrowOverhead);
        bytes += (long long)s.n_kv * q.len * s.key_bytes;
    }
    const bool narrow = cost && (!chunks || bytes > kWideBytes);
    plan->stream = narrow && bytes > kStreamBytes;
    // the rows that the narrow kernel takes
    auto is_narrow = [&](const PagedSeq& q) { return narrow && (long long)q.n_new * s.group <= kNarrowRows; };
    int counter = 0;
    if (narrow) {
        first.push_back(0);
        // The least share that the workgroups can take all of: cuts cost more than the columns alone,
        // so an even share of these is tried first and then grown.
        long long share = std::max<long long>((cost + s.narrow_wgs - 1) / s.narrow_wgs, kNarrowLeast + kNarrowOverhead);
        if (longest <= kNarrowWhole) share = std::max<long long>(share, longest + kNarrowOverhead);
        // what a workgroup takes of a column's `left` tiles with `room` to go; 0: nothing
        auto piece = [](long long room, int left) {
            const long long take = room - kNarrowOverhead;
            return take < std::min(kNarrowLeast, left) ? 0 : left - take < kNarrowLeast ? left : (int)take;
        };
        for (;; share += share / 64 + 1) {
            int need = 1;
            long long room = share;
            for (const PagedSeq& q : plan->seqs) {
                if (!q.n_new || !is_narrow(q)) continue;
                const int tiles = (q.len + kNarrowKeys - 1) / kNarrowKeys;
                for (int kvh = 0; kvh < s.n_kv && need <= s.narrow_wgs; kvh++)
                    for (int t = 0; t < tiles;) {
                        const int take = piece(room, tiles - t);
                        if (!take) {
                            need++;
                            room = share;
                        }
                        t += take;
                        room -= take ? take + kNarrowOverhead : 0;
                    }
            }
            if (need <= s.narrow_wgs) break;
        }
        int slot = 0;
        long long room = share;
        for (const PagedSeq& q : plan->seqs) {
            if (!q.n_new || !is_narrow(q)) continue;
            const int tiles = (q.len + kNarrowKeys - 1) / kNarrowKeys;
            for (int kvh = 0; kvh < s.n_kv; kvh++) {
                const size_t begin = items.size();
                for (int t = 0; t < tiles;) {
                    const int take = piece(room, tiles - t);
                    if (!take) {  // no room for a piece: the next workgroup
                        first.push_back((int)items.size());
                        room = share;
                        continue;
                    }
                    items.push_back({q.row0, q.n_new * s.group, q.len - q.n_new, q.table, kvh, 0, t, t + take, 0, 0, 1, 0});
                    t += take;
                    room -= take + kNarrowOverhead;
                }
                const int parts = (int)(items.size() - begin);
                if (parts > 1) {
                    for (int p = 0; p < parts; p++) {
                        PagedItem& it = items[begin + p];
                        it.slot0 = slot;
                        it.part = p;
                        it.parts = parts;
                        it.counter = counter;
                    }
                    slot += parts;
                    counter++;
                }
            }
        }
        first.push_back((int)items.size());
        for (size_t w = 0; w + 1 < first.size(); w++) {
            plan->runs.push_back({first[w + 1] - first[w], (int)plan->rest.size(), {0, 0}, items[first[w]]});
            plan->rest.insert(plan->rest.end(), items.begin() + first[w] + 1, items.begin() + first[w + 1]);
        }
    }
    // wide
    struct Block {
        int seq, r0, tiles;
    };
    std::vector<Block> blocks;
    long long total = 0, full = 0;
    for (const PagedSeq& q : plan->seqs)
        if (q.n_new && !is_narrow(q)) full += ((long long)q.n_new * s.group + s.wide_rows - 1) / s.wide_rows;
    plan->wide_rows = full * s.n_kv < s.wide_wgs ? s.least_rows : s.wide_rows;
    for (size_t i = 0; i < plan->seqs.size(); i++) {
        const PagedSeq& q = plan->seqs[i];
        const long long rows = (long long)q.n_new * s.group;
        if (!rows || is_narrow(q)) continue;
        for (int r0 = 0; r0 < rows; r0 += plan->wide_rows) {
            const int last = (int)std::min<long long>(rows, (long long)r0 + plan->wide_rows) - 1;
            const int keys = q.len - q.n_new + last / s.group + 1;
            const int tiles = (keys + s.wide_keys - 1) / s.wide_keys;
            blocks.push_back({(int)i, r0, tiles});
            total += tiles;
        }
    }
    if (blocks.empty()) return;
    std::stable_sort(blocks.begin(), blocks.end(), [](const Block& a, const Block& b) { return a.tiles > b.tiles; });
    // tiles of a part: an even share of all
    const long long target = std::max<long long>((total * s.n_kv + s.wide_wgs - 1) / s.wide_wgs, kWideLeast / s.wide_keys);
    counter = 0;
    int slot = 0;
    for (const Block& b : blocks) {
        const PagedSeq& q = plan->seqs[b.seq];
        // to the nearest: the cut blocks' parts are at most 4/3 of wide_wgs in all
        const int parts = (int)std::max<long long>(1, (b.tiles + target / 2) / target);
        for (int p = 0; p < parts; p++)
            for (int kvh = 0; kvh < s.n_kv; kvh++) {
                PagedItem it = {q.row0, q.n_new * s.group, q.len - q.n_new, q.table, kvh, b.r0,
                                (int)((long long)b.tiles * p / parts), (int)((long long)b.tiles * (p + 1) / parts), 0, p, parts, 0};
                if (parts > 1) {
                    it.slot0 = slot + kvh * parts;
                    it.counter = counter + kvh;
                }
                plan->wide.push_back(it);
            }
        if (parts > 1) {
            slot += parts * s.n_kv;
            counter += s.n_kv;
        }
    }
}

}  // namespace pqa
