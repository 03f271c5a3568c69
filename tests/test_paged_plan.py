"""The paged batch's checks and its cutting into work items (picolm_qwen_amd/csrc/pqa_paged_plan.h),
built on the CPU with g++: over random batches every key tile of every block of rows is one item's,
cut blocks have consecutive parts with slots and a counter of their own, and nothing exceeds
what the batch allocates; every contradiction in the caller's arrays is refused."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>

#include "pqa_paged_plan.h"

using namespace pqa;

static PagedShape shape(int page, int group, int n_kv, int wgs, int rows, int keys) {
    PagedShape s{};
    s.n_pages = 40000;
    s.page_size = page;
    s.group = group;
    s.n_kv = n_kv;
    s.max_pos = 0;
    s.narrow_wgs = wgs;
    s.wide_wgs = 2 * wgs;
    s.wide_rows = rows;
    s.least_rows = 64;
    s.wide_keys = keys;
    s.max_seqs = 96;
    s.max_tokens = 8192;
    s.max_seq_pages = 9000;
    s.key_bytes = 512;
    return s;
}

#define CHECK(c)                                                        \
    do {                                                                \
        if (!(c)) {                                                     \
            std::printf("trial %d line %d: %s\n", trial, __LINE__, #c); \
            return 1;                                                   \
        }                                                               \
    } while (0)

static int check(int trial, const PagedShape& s, const PagedPlan& p, const std::vector<PagedItem>& items, bool wide) {
    const int rows = wide ? p.wide_rows : kNarrowRows, keys = wide ? s.wide_keys : kNarrowKeys;
    const int slots = wide ? paged_wide_slots(s) : paged_narrow_slots(s), counters = wide ? s.wide_wgs : s.narrow_wgs;
    std::map<std::tuple<int, int, int>, std::vector<PagedItem>> blocks;
    for (const PagedItem& it : items) blocks[{it.table, it.kvh, it.r0}].push_back(it);
    std::set<int> used_slots, used_counters;
    size_t want = 0, n_blocks = 0;
    for (const PagedSeq& q : p.seqs) {
        const long long r = (long long)q.n_new * s.group;
        if (!q.n_new || (r > kNarrowRows || p.runs.empty()) != wide) continue;
        for (int kvh = 0; kvh < s.n_kv; kvh++)
            for (int r0 = 0; r0 < r; r0 += rows) {
                n_blocks++;
                auto b = blocks.find({q.table, kvh, r0});
                CHECK(b != blocks.end());
                auto& v = b->second;
                std::sort(v.begin(), v.end(), [](const PagedItem& x, const PagedItem& y) { return x.part < y.part; });
                want += v.size();
                const int last = (int)std::min<long long>(r, (long long)r0 + rows) - 1;
                const int seen = q.len - q.n_new + last / s.group + 1, tiles = (seen + keys - 1) / keys;
                int t = 0;
                for (size_t i = 0; i < v.size(); i++) {
                    CHECK(v[i].row0 == q.row0 && v[i].rows == r && v[i].hist == q.len - q.n_new);
                    CHECK(v[i].t0 == t && v[i].t1 > t);
                    t = v[i].t1;
                    CHECK(v[i].part == (int)i && v[i].parts == (int)v.size());
                    if (v.size() > 1) {
                        CHECK(v[i].slot0 == v[0].slot0 && v[i].counter == v[0].counter);
                        CHECK(v[i].slot0 >= 0 && v[i].slot0 + (int)i < slots);
                        CHECK(used_slots.insert(v[i].slot0 + (int)i).second);
                    }
                }
                CHECK(t == tiles);
                if (v.size() > 1) {
                    CHECK(v[0].counter >= 0 && v[0].counter < counters);
                    CHECK(used_counters.insert(v[0].counter).second);
                }
            }
    }
    CHECK(want == items.size());
    const size_t most = wide ? ((size_t)s.max_tokens * s.group / s.wide_rows + s.max_seqs) * s.n_kv + 4 * s.wide_wgs
                             : (size_t)s.max_seqs * s.n_kv + s.narrow_wgs;
    CHECK(items.size() <= most);
    return 0;
}

int main() {
    std::mt19937 rng(7);
    auto draw = [&](double lo, double hi) {
        return (int)std::lround(std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi))(rng)));
    };
    for (int trial = 0; trial < 300; trial++) {
        const int page = 16 << (rng() % 5), groups[] = {1, 2, 4, 7, 8, 16, 17, 32}, kvs[] = {1, 2, 3, 8, 32};
        PagedShape s = shape(page, groups[rng() % 8], kvs[rng() % 5], trial % 3 ? 256 : trial % 2 ? 512 : 3, trial % 2 ? 64 : 128,
                             trial % 5 ? 64 : 32);
        const int n = trial % 7 ? draw(1, 96) : trial % 2;
        std::vector<int> n_new, len, pages;
        const int stride = s.max_seq_pages;
        int next = 0, left = s.max_tokens;
        for (int i = 0; i < n; i++) {
            const int l = draw(1, i % 4 ? 3000 : 60000 / (1 + n / 8));
            int m = rng() % 3 ? 1 : rng() % 5 ? draw(1, 1500) : 0;
            m = std::min({m, l, left});
            left -= m;
            n_new.push_back(m);
            len.push_back(l);
        }
        pages.assign((size_t)std::max(n, 1) * stride, -1);
        for (int i = 0; i < n; i++)
            for (int j = 0; j < (len[i] + page - 1) / page; j++) pages[(size_t)i * stride + j] = next++;
        s.n_pages = std::max(next, 1);
        PagedPlan p;
        std::string why;
        const PagedFault f = paged_check(s, n, n_new.data(), len.data(), pages.data(), stride, &p, &why);
        if (f != PagedFault::none) std::printf("%s\n", why.c_str());
        CHECK(f == PagedFault::none);
        CHECK((int)p.tokens.size() == p.n_tok && p.n_tok == s.max_tokens - left);
        for (const PagedSeq& q : p.seqs)
            for (int i = 0; i < q.n_new; i++) {
                const PagedToken& t = p.tokens[q.row0 + i];
                CHECK(t.table == q.table && t.pos == q.len - q.n_new + i && t.nth == i && t.left == q.n_new - i);
            }
        CHECK(p.touched.size() <= std::min((size_t)s.max_tokens, (size_t)2 * s.max_seqs + s.max_tokens / page));
        for (const PagedTouched& t : p.touched) CHECK(t.used >= 1 && t.used <= page);
        paged_items(s, &p);
        CHECK((int)p.runs.size() <= s.narrow_wgs);
        std::vector<PagedItem> items;
        long long tiles = 0, most = 0;
        for (const PagedRun& r : p.runs) {
            CHECK(r.count >= 1 && r.rest >= 0 && (size_t)(r.rest + r.count - 1) <= p.rest.size());
            long long mine = 0;
            for (int i = 0; i < r.count; i++) {
                const PagedItem& it = i ? p.rest[r.rest + i - 1] : r.first;
                items.push_back(it);
                mine += it.t1 - it.t0 + kNarrowOverhead;
            }
            tiles += mine;
            most = std::max(most, mine);
        }
        CHECK(items.size() == p.rest.size() + p.runs.size());
        // no workgroup has much more than its share of the tiles (or one whole short column)
        CHECK(most <= tiles / s.narrow_wgs * 1.1 + 2 * (kNarrowOverhead + kNarrowLeast) + kNarrowWhole);
        if (check(trial, s, p, items, false) || check(trial, s, p, p.wide, true)) return 1;
        // what pqa_batch_create holds for the wide kernel's partials of this very batch
        size_t blocks = 0, cut = 0;
        int longest = 0, rows = 0;
        for (int i = 0; i < n; i++) {
            longest = std::max(longest, len[i]);
            rows = std::max(rows, n_new[i] * s.group);
        }
        if ((long long)p.n_tok * s.group > kNarrowRows) blocks = (size_t)p.n_tok * s.group / s.least_rows + std::min(n, p.n_tok);
        for (const PagedItem& it : p.wide) cut = std::max(cut, it.parts > 1 ? (size_t)it.slot0 + it.parts : 0);
        CHECK(cut <= blocks * s.n_kv * (longest / kWideLeast + 1));
    }

    // refusals
    const int trial = -1;
    PagedShape s = shape(16, 4, 2, 256, 128, 64);
    s.n_pages = 10;
    s.max_seqs = 3;
    s.max_tokens = 20;
    s.max_seq_pages = 4;
    s.max_pos = 60;
    PagedPlan p;
    std::string why;
    auto go = [&](std::vector<int> n_new, std::vector<int> len, std::vector<int> pages, int stride) {
        return paged_check(s, (int)n_new.size(), n_new.data(), len.data(), pages.data(), stride, &p, &why);
    };
    CHECK(go({1, 1}, {17, 5}, {0, 1, 2, -1}, 2) == PagedFault::none);
    CHECK(go({}, {}, {}, 0) == PagedFault::none && p.n_tok == 0);
    CHECK(go({1, 1, 1, 1}, {1, 1, 1, 1}, {0, 1, 2, 3}, 1) == PagedFault::argument);   // too many sequences
    CHECK(go({-1}, {5}, {0}, 1) == PagedFault::argument);
    CHECK(go({6}, {5}, {0}, 1) == PagedFault::argument);                              // more new tokens than positions
    CHECK(go({1}, {-3}, {0}, 1) == PagedFault::argument);
    CHECK(go({1}, {17}, {0}, 1) == PagedFault::range);                                // list too short
    CHECK(go({1}, {61}, {0, 1, 2, 3}, 4) == PagedFault::range);                       // past the rotation's tables
    s.max_pos = 0;
    CHECK(go({1}, {65}, {0, 1, 2, 3, 4}, 5) == PagedFault::range);                    // past the batch's max_len
    CHECK(go({21}, {21}, {0, 1}, 2) == PagedFault::range);                            // too many tokens
    CHECK(go({1}, {2147483647}, {0, 1}, 2) == PagedFault::range);
    CHECK(go({1}, {17}, {0, 10}, 2) == PagedFault::argument);                         // page outside the pool
    CHECK(go({1}, {17}, {-1, 1}, 2) == PagedFault::argument);
    CHECK(go({1}, {17}, {1, 1}, 2) == PagedFault::argument);                          // its own page twice, one written
    CHECK(go({1, 1}, {5, 5}, {3, 3}, 1) == PagedFault::argument);                     // two sequences write one page
    CHECK(go({1, 1}, {5, 17}, {3, -1, 3, 4}, 2) == PagedFault::argument);             // one writes what another reads
    CHECK(go({1, 1}, {17, 5}, {3, 4, 3, -1}, 2) == PagedFault::argument);             // the same, the reader first
    CHECK(go({1, 1}, {17, 17}, {3, 4, 3, 5}, 2) == PagedFault::none);                 // a shared prompt, read only
    CHECK(go({0, 1}, {17, 17}, {3, 4, 3, 5}, 2) == PagedFault::none);
    CHECK(go({0, 1}, {0, 17}, {-1, -1, 3, 5}, 2) == PagedFault::none);                // an empty sequence
    std::printf("ok\n");
    return 0;
}
"""


def test_plans_cover_every_tile_once_and_bad_batches_are_refused(tmp_path):
    src = tmp_path / "plan.cpp"
    src.write_text(SRC)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    "-I" + os.path.join(ROOT, "picolm_qwen_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", (out.stdout, out.stderr[-3000:])
