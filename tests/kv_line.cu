// Host-only checks of the index logic behind attention over a paged cache (gpt_b200/csrc/kv_pages.cuh): built and run by tests/test_kv_pages_cpu.py, no GPU.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv_pages.cuh"

using namespace gptb200::kvp;

#define REQUIRE(c)                                                        \
    do {                                                                  \
        if (!(c)) {                                                       \
            std::printf("%s:%d: %s (case %d)\n", __FILE__, __LINE__, #c, g_case); \
            std::exit(1);                                                 \
        }                                                                 \
    } while (0)

static int g_case = 0;

static void divisions()
{
    std::mt19937 rng(1);
    for (uint32_t by : {1u, 2u, 3u, 4u, 5u, 6u, 7u, 8u, 12u, 20u, 24u, 96u, 100u, 255u, 256u, 1000u, 65537u, 1000003u}) {
        const Divisor d = divisor(by);
        for (int n : {0, 1, 2, 2147483647, 2147483646, 1 << 30}) REQUIRE(d.divide(n) == int(n / by));
        for (int i = 0; i < 20000; ++i) {
            const int n = int(rng() & 0x7fffffffu) >> (rng() % 31);
            REQUIRE(d.divide(n) == int(n / by));
        }
    }
}

struct Case {
    std::vector<int> starts, lengths, table;
    Attention a{};
    int status = 0;
    void point()
    {
        a.batch.row_starts = starts.data();
        a.batch.lengths = lengths.data();
        a.batch.table = table.data();
        a.batch.status = &status;
    }
};

// Every block of every tile goes to exactly one block of the grid, parts of a tile to neighbours that know one another; at most one part of a block begins before it
// and one goes on behind it.
static void line(std::mt19937 &rng)
{
    Case c;
    const int sequences = 1 + rng() % 9, share = 1 + rng() % 9;
    c.starts = {0};
    int longest = 1;
    for (int s = 0; s < sequences; ++s) {
        const int length = rng() % (rng() % 4 ? 300 : 5000), n = rng() % 5 == 0 ? 0 : rng() % 3 ? 1 : 1 + rng() % 200;
        c.starts.push_back(c.starts.back() + n);
        c.lengths.push_back(length);
        longest = std::max(longest, length);
    }
    Attention &a = c.a;
    a.pages = {nullptr, nullptr, 100, 3 + int(rng() % 5), 1 + int(rng() % 4), 64};
    a.share = share;
    a.shares = divisor(share);
    a.heads = share * a.pages.kv_heads;
    a.window = rng() % 2 ? 1 + rng() % 400 : 0;
    a.sinks = a.window ? rng() % 90 : 0;
    a.batch.sequences = sequences;
    a.batch.rows = c.starts.back() + rng() % 3;
    a.batch.table_pitch = (longest >> a.pages.page_shift) + 1;
    a.batch.capacity = a.batch.table_pitch << a.pages.page_shift;
    c.table.assign(size_t(sequences) * a.batch.table_pitch, 0);
    c.point();
    const int shapes[5][2] = {{8, 64}, {16, 64}, {256, 128}, {1, 64}, {16, 32}};
    const int *shape = shapes[rng() % 5];
    const Cut cut = {shape[0], shape[1], 1 + int(rng() % 2), 3 + int(rng() % 4)};
    struct Tile {
        int s, g, t;
        long long first;
        KeyBlocks blocks;
    };
    std::vector<Tile> tiles;
    long long total = 0, added = 0;
    for (int s = 0; s < sequences; ++s) {
        const Sequence q = sequence_of(a.batch, s);
        added += blocks_of(a, q, cut) * a.pages.kv_heads;
        for (int g = 0; g < a.pages.kv_heads; ++g)
            for (int t = 0; t < tiles_of(a, q, cut.tile_rows); ++t) {
                const KeyBlocks b = tile_blocks(a, q, t, cut.tile_rows, cut.keys);
                tiles.push_back({s, g, t, total, b});
                total += cut.lead + b.count;
                // the blocks hold every key that a row of the tile sees, none twice
                std::vector<int> held(longest + 2 * cut.keys + 1, 0);
                for (int i = 0; i < b.count; ++i)
                    for (int k = 0; k < cut.keys; ++k) {
                        const int key = block_key(b, i, cut.keys) + k;
                        if (key < int(held.size())) held[key]++;
                    }
                for (int p = t * cut.tile_rows; p < std::min((t + 1) * cut.tile_rows, q.count * share); p += 1 + (p % 7)) {
                    const int position = q.pos0 + p / share;
                    for (int key = 0; key <= position; ++key)
                        if (visible(a, key, position)) REQUIRE(held[key] == 1);
                }
            }
    }
    REQUIRE(added == total && c.status == 0);
    if (total == 0) return;
    const int grid = 1 + rng() % (rng() % 3 ? 40 : 500);
    std::vector<std::vector<int>> owner(tiles.size());
    for (size_t i = 0; i < tiles.size(); ++i) owner[i].assign(tiles[i].blocks.count, -1);
    for (int b = 0; b < grid; ++b) {
        Range r = range_of(total, b, grid, cut);
        if (r.begin >= r.end) continue;
        size_t at_tile = 0;
        while (tiles[at_tile].first + cut.lead + tiles[at_tile].blocks.count <= r.begin) ++at_tile;
        Place p;
        p.s = tiles[at_tile].s;
        p.g = tiles[at_tile].g;
        p.tile = tiles[at_tile].t;
        p.q = sequence_of(a.batch, p.s);
        p.tiles = tiles_of(a, p.q, cut.tile_rows);
        p.blocks = tiles[at_tile].blocks;
        p.off = int(r.begin - tiles[at_tile].first);
        if (!settle(a, cut, r, p) || !takes(r, p, r.begin, cut)) continue;
        int heads = 0, tails = 0;
        for (long long at = r.begin;;) {
            at_tile = 0;
            while (tiles[at_tile].s != p.s || tiles[at_tile].g != p.g || tiles[at_tile].t != p.tile) ++at_tile;
            const Tile &t = tiles[at_tile];
            REQUIRE(at - p.off == t.first);
            const Part part = part_of(p, r, at, cut);
            REQUIRE(part.blocks > 0 && part.from + part.blocks <= t.blocks.count);
            for (int i = 0; i < part.blocks; ++i) {
                REQUIRE(owner[at_tile][part.from + i] == -1);
                owner[at_tile][part.from + i] = b;
            }
            if (!part.whole) {
                REQUIRE(part.b0 <= b && b <= part.b1 && part.b0 < part.b1 && part.tail == (b == part.b0));
                (part.tail ? tails : heads)++;
            }
            at += part.places;
            if (!advance(a, r, p, at, cut)) break;
        }
        REQUIRE(heads <= 1 && tails <= 1);
    }
    for (size_t i = 0; i < tiles.size(); ++i) {
        int first = owner[i].front(), last = owner[i].back();
        REQUIRE(first >= 0);
        for (size_t k = 1; k < owner[i].size(); ++k) REQUIRE(owner[i][k] == owner[i][k - 1] || owner[i][k] == owner[i][k - 1] + 1);
        // who shares the tile knows it
        Range r = range_of(total, first, grid, cut);
        Place p{};
        p.blocks = tiles[i].blocks;
        p.off = 0;
        const Part part = part_of(p, r, tiles[i].first, cut);
        REQUIRE(part.whole == (first == last));
        if (!part.whole) REQUIRE(part.b0 == first && part.b1 == last);
    }
}

// Whatever the arrays hold, rows stay inside the tensors, positions inside the table and pages inside the pool; and it is reported.
static void nonsense(std::mt19937 &rng)
{
    Case c;
    const int sequences = 1 + rng() % 6;
    auto any = [&] { return rng() % 3 ? int(rng() % 200) - 60 : int(rng()); };
    for (int s = 0; s <= sequences; ++s) c.starts.push_back(any());
    for (int s = 0; s < sequences; ++s) c.lengths.push_back(any());
    Attention &a = c.a;
    a.pages = {nullptr, nullptr, 7, 4, 2, 64};
    a.share = 3;
    a.shares = divisor(3);
    a.window = rng() % 2 ? 1 + rng() % 50 : 0;
    a.sinks = rng() % 9;
    a.batch.sequences = sequences;
    a.batch.rows = rng() % 150;
    a.batch.table_pitch = 4;
    a.batch.capacity = 64;
    for (int i = 0; i < 4 * sequences; ++i) c.table.push_back(any());
    c.point();
    bool fits = true;
    for (int s = 0; s < sequences; ++s) {
        const Sequence q = sequence_of(a.batch, s);
        REQUIRE(q.row0 >= 0 && q.count >= 0 && q.row0 + q.count <= a.batch.rows && q.pos0 + q.count <= a.batch.capacity);
        fits = fits && c.starts[s] >= 0 && c.starts[s] <= c.starts[s + 1] && c.starts[s + 1] <= a.batch.rows && c.lengths[s] >= 0 && c.lengths[s] <= 64;
        for (int t = 0; t < tiles_of(a, q, 16); ++t) {
            const KeyBlocks b = tile_blocks(a, q, t, 16, 64);
            REQUIRE(b.count >= 1 && block_key(b, b.count - 1, 64) < 64);
        }
    }
    REQUIRE((c.status == 0) == fits);
    for (int s = 0; s < sequences; ++s)
        for (int position = 0; position < 64; ++position) {
            c.status = 0;
            const int page = page_of(a.batch, a.pages, s, position), there = c.table[4 * s + position / 16];
            REQUIRE(page >= -1 && page < 7 && (page == -1) == (there < 0 || there >= 7) && (c.status != 0) == (page == -1));
        }
}

int main()
{
    divisions();
    std::mt19937 rng(7);
    for (g_case = 0; g_case < 3000; ++g_case) line(rng);
    for (g_case = 0; g_case < 2000; ++g_case) nonsense(rng);
    std::printf("ok\n");
}
