"""What the decode attention's look-ahead reads of block tables and lengths, which no result shows: the kernel's own lines, compiled for the
host around tables that check every read."""
import re
import shutil
import subprocess
from pathlib import Path

KERNEL = Path(__file__).resolve().parent.parent / "nano-vllm-moe_b200" / "csrc" / "paged_attention.cu"

HARNESS = r"""
#include <stdint.h>
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#define __device__
#define __forceinline__ inline
#define __host__
using std::min;
constexpr int kBlock = 16;

struct Slice {                                  // of a caller's memory
    const std::vector<int>* all;
    int64_t at;
    Slice operator+(int64_t n) const { return {all, at + n}; }
};
long long outside = 0, read = 0;
int ld_dep(Slice s) {
    ++read;
    if (s.at >= 0 && s.at < (int64_t)s.all->size()) return (*s.all)[s.at];
    ++outside;
    return -7;
}
struct ByDivision { int d; int quotient(int n) const { return n / d; } };
struct AttnArgs {
    struct { int kv_heads, block_size; } c;
    Slice tables, lens;
    int64_t ld_tables, max_pages;
    int batch;
    ByDivision by_page, by_parts;
};
struct Seen { int b, len, token0, pages, behind, at_page, off; };         // of a block of 16 tokens, in one lane
int64_t quotient(int64_t n, int64_t d) { return n / d; }

@FUNCTIONS@

// One lane of a warp that has `span` places of the list from `begin` on: its tiles, with what the lane has at hand for them.
template <int kTile>
std::vector<Seen> walk(const AttnArgs& a, int lane, int parts, int64_t begin, int span) {
    auto tiles_of = [](int len) { return tiles_in<kTile>(len); };
    const int64_t most64 = a.max_pages * a.c.block_size, most = most64 < 0x7fffff00 ? most64 : 0x7fffff00;
    struct Found { int b, len; int64_t inside; };
    const bool apart = false;
    const Found own = {};
    const int own_segment = 0, before = 0, mine = 0, places_of = 0;
    auto find = [&](int, int, int, int64_t place) {
        for (int b = 0;; ++b) {
            const int len = within((*a.lens.all)[b], most);
            const int64_t all = (int64_t)(tiles_of(len) + kBegin) * a.c.kv_heads * parts;
            if (place < all) return Found{b, len, place};
            place -= all;
        }
    };
    std::vector<Seen> seen;
@PAGES@
@BEGIN@
@NEXT_TILE@
    while (in.place < span) {
        for (int h = 0; h < kTile / kBlock; ++h) {
@NEXT_BLOCK@
            seen.push_back({in.b, in.len, in.t * kTile + h * kBlock, pages, pages_behind, at_page, off16});
        }
        next_tile();
    }
    return seen;
}

int main() {
    std::mt19937 rng(1);
    auto pick = [&](auto... x) { const std::vector<int> v = {x...}; return v[rng() % v.size()]; };
    int bad = 0;
    for (int i = 0; i < 3000; ++i) {
        const int batch = pick(1, 1, 2, 3, 7), heads = pick(1, 2, 4), parts = pick(1, 1, 2, 3), size = pick(1, 3, 5, 8, 16, 17, 24, 32, 256);
        const int pages = pick(0, 1, 2, 31, 32, 33, 47, 63, 64, 65, 96, 130), most = pages * size;
        const bool wide = rng() % 2;
        std::vector<int> lens, table;
        int64_t total = 0;
        for (int b = 0; b < batch; ++b) {
            lens.push_back(rng() % 4 == 0 ? most : (int)(rng() % (most + 9)) - 4);
            const int n = within(lens[b], most);
            total += (int64_t)((wide ? tiles_in<32>(n) : tiles_in<16>(n)) + kBegin) * heads * parts;
        }
        for (int e = 0; e < batch * pages; ++e) table.push_back((int)(rng() % 1000000));
        const AttnArgs a = {{heads, size}, {&table, 0}, {&lens, 0}, pages, pages, batch, {size}, {parts}};
        const int64_t share = total / pick(1, 2, 5, 40) + 1;
        const long long before = outside;
        long long wrong = 0;
        for (int64_t from = 0; from < total; from += share) {
            std::vector<Seen> lanes[32];
            for (int lane = 0; lane < 32; ++lane)
                lanes[lane] = wide ? walk<32>(a, lane, parts, from, (int)min(share, total - from)) : walk<16>(a, lane, parts, from, (int)min(share, total - from));
            for (size_t k = 0; k < lanes[0].size(); ++k) {
                const Seen& s = lanes[0][k];
                for (int r = 0; r < kBlock && s.token0 + r < s.len; ++r) {
                    const int token = s.token0 + r, page = (s.off + r) / size, which = s.at_page + page;
                    const int got = which < 32 ? lanes[which][k].pages : which < 64 ? lanes[which - 32][k].behind : -1;
                    wrong += got != table[s.b * pages + token / size] || s.off + r - page * size != token % size;
                }
            }
        }
        if ((wrong || outside != before) && ++bad <= 5)
            printf("batch %d, %d key heads, %d parts, pages of %d, %d entries per table, tiles of %d: %lld tokens on a wrong page, %lld reads outside\n", batch, heads, parts, size,
                   pages, wide ? 32 : 16, wrong, outside - before);
    }
    printf("%d of 3000 batches are wrong, %lld reads\n", bad, read);
    return bad != 0;
}
"""


def cut(text, first, last=None):
    """The line that begins with `first`, and all up to the next one that begins with `last`."""
    rest = rf".*?^[ ]*{re.escape(last)}[^\n]*" if last else r"[^\n]*"
    found = re.search(rf"^[ ]*{re.escape(first)}{rest}\n", text, re.S | re.M)
    assert found, (first, last)
    return found.group(0)


def test_the_walk_over_the_tables_reads_only_what_they_hold(tmp_path):
    text = KERNEL.read_text()
    parts = {
        "FUNCTIONS": cut(text, "constexpr int kBegin") + cut(text, "__device__ __forceinline__ int within(") + "template <int kTile>\n"
        + cut(text, "__device__ __forceinline__ int tiles_in("),
        "PAGES": cut(text, "const int page_size = a.c.block_size", "auto pages_in"),
        "BEGIN": cut(text, "struct Place {", "// copies: lane ->"),
        "NEXT_TILE": cut(text, "auto next_tile = [&] {", "};"),
        "NEXT_BLOCK": cut(text, "if (page_at - page_base >= 32) {", "page_off +="),
    }
    source = HARNESS
    for name, code in parts.items():
        source = source.replace(f"@{name}@", code)
    (tmp_path / "walk.cpp").write_text(source)
    subprocess.run([shutil.which("g++") or "g++", "-O1", "-std=c++17", "-o", str(tmp_path / "walk"), str(tmp_path / "walk.cpp")], check=True, timeout=300)
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    # ... and the kernel reads tables nowhere else
    plain = re.sub(r"//[^\n]*", "", text)
    assert plain.count("a.tables") == 1 and "a.tables" in parts["BEGIN"]
