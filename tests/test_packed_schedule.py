"""How a ragged batch is cut up (flint_b200/csrc/packed_schedule.h), checked on the CPU.

The header is plain C++. A small program goes through random batches, cuts each as the kernel's CTAs do, and
requires that every (sequence, K/V head, tile, key tile) is worked on exactly once, that a key tile a
token sees is never left out, that the records name exactly the tiles that were split with their parts in
order, and that no CTA gets much more than its share.
"""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).parent.parent / "flint_b200" / "csrc"

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>
#include "packed_schedule.h"
using namespace fb;
#define NEED(x) do { if (!(x)) { std::printf("line %d: %s (trial %d)\n", __LINE__, #x, trial); return 1; } } while (0)

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int a, int b) { return static_cast<int>(a + rng() % (b - a + 1)); };
    for (int trial = 0; trial < 3000; ++trial) {
        const int count = pick(1, trial % 3 ? 6 : 60), kv_heads = pick(1, 5), log_tokens = pick(0, 7);
        const int most = trial % 5 ? pick(1, 40) : 296, least = pick(1, 4);
        std::vector<Sequence> all;
        int first = pick(0, 3);
        for (int s = 0; s < count; ++s) {
            const int tokens = trial % 4 == 0 ? 1 : pick(0, 5) == 0 ? 0 : pick(1, trial % 7 ? 300 : 2000);
            const int kind = pick(0, 5);
            const int keys = kind == 0 ? pick(0, tokens) : kind < 3 ? tokens : tokens + pick(0, trial % 11 ? 500 : 20000);
            all.push_back({first, tokens, keys});
            first += tokens;
        }
        auto get = [&](int s) { return all.at(s); };
        // Lengths against a plain sum, tile by tile.
        long long total = 0;
        for (const auto& q : all) {
            long long sum = 0;
            for (int i = 0; i < tile_count(q.count, log_tokens); ++i) {
                NEED(tiles_before(q.before(), log_tokens, i) == sum);
                const int last = std::min((i + 1) << log_tokens, q.count);
                const int sees = std::max(0, q.before() + last);
                NEED(key_tiles(q.before(), q.count, log_tokens, i) == std::max(1, (sees + 127) / 128));
                sum += key_tiles(q.before(), q.count, log_tokens, i) + kTileEnds;
            }
            NEED(head_length(q.before(), q.count, log_tokens) == sum);
            total += sum * kv_heads;
        }
        const int parts = part_count(total, most, least);
        NEED(parts <= most && (total == 0 || parts >= 1));
        auto cut = [&](int k) {
            const long long at = cut_place(total, parts, k);
            if (at == total) {
                return Cut{total, count, 0, 0, 0};
            }
            long long begins = 0;
            for (int s = 0;; ++s) {
                const long long length = head_length(all[s].before(), all[s].count, log_tokens);
                if (at < begins + length * kv_heads) {
                    return cut_at(at, at - begins, s, all[s].before(), all[s].count, log_tokens, length,
                                  cut_tolerance(total, parts));
                }
                begins += length * kv_heads;
            }
        };
        std::map<std::tuple<int, int, int>, std::vector<std::tuple<int, int, int>>> done;   // (from, to, cta)
        std::vector<Record> records;
        for (int k = 0; k < parts; ++k) {
            const Cut lo = cut(k), hi = cut(k + 1);
            NEED(lo.at <= hi.at && (k > 0 || lo.at == 0) && (k + 1 < parts || hi.at == total));
            NEED(hi.at - lo.at <= total / parts + 1 + 2 * cut_tolerance(total, parts));
            records.push_back(make_record(get, log_tokens, lo, hi));
            Walk walk;
            Piece piece;
            walk.begin(get, lo, hi.at);
            int pieces = 0;
            bool tail = false;
            while (walk.next(get, count, kv_heads, log_tokens, piece)) {
                const Sequence& q = all[piece.index];
                NEED(piece.tokens >= 1 && piece.first_token + piece.tokens <= q.count && piece.head < kv_heads);
                NEED(0 <= piece.from && piece.from < piece.to && piece.to <= piece.tiles);
                NEED(!tail);
                if (piece.from > 0) {
                    NEED(pieces == 0 && records[k].head_part == (piece.to < piece.tiles ? 2 : 1));
                } else {
                    NEED(pieces > 0 || records[k].head_part == 0);
                }
                tail = piece.to < piece.tiles;
                if (tail && piece.from == 0) {
                    const Record& r = records[k];
                    NEED(r.tail_part == 1 && r.first_row == q.first + piece.first_token && r.tokens == piece.tokens);
                    NEED(r.kv_head == piece.head && r.position == piece.position());
                }
                done[{piece.index, piece.head, piece.first_token}].push_back({piece.from, piece.to, k});
                ++pieces;
            }
            if (records[k].tail_part) {
                NEED(tail);
            }
            if (records[k].head_part) {
                NEED(pieces > 0);
            }
        }
        size_t tiles = 0;
        for (int s = 0; s < count; ++s) {
            tiles += static_cast<size_t>(tile_count(all[s].count, log_tokens)) * kv_heads;
        }
        NEED(done.size() == tiles);
        for (const auto& [tile, list] : done) {
            const auto& q = all[std::get<0>(tile)];
            int at = 0;
            for (size_t i = 0; i < list.size(); ++i) {
                const auto& [from, to, cta] = list[i];
                NEED(from == at);
                at = to;
                if (list.size() > 1) {
                    // The join starts at the first part's CTA and goes on while a record says so.
                    if (i == 0) {
                        NEED(records[cta].tail_part == 1);
                    } else {
                        NEED(cta == std::get<2>(list[i - 1]) + 1);
                        NEED(records[cta].head_part == (i + 1 < list.size() ? 2 : 1));
                    }
                }
            }
            NEED(at == key_tiles(q.before(), q.count, log_tokens, std::get<2>(tile) >> log_tokens));
        }
    }
    // The largest sizes: no 32-bit overflow.
    const int trial = -1;
    NEED(head_length(0, 1 << 24, 0) > (1LL << 40));
    NEED(head_length((1 << 26) - 1, 1, 0) == (1 << 19) + kTileEnds);
    NEED(key_tiles((1 << 26) - (1 << 24), 1 << 24, 7, (1 << 17) - 1) == 1 << 19);
    return 0;
}
"""


def test_every_key_tile_is_worked_on_once(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "schedule.cpp").write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(tmp_path / "schedule.cpp"), "-o", str(tmp_path / "schedule")], check=True)
    result = subprocess.run([str(tmp_path / "schedule")], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout + result.stderr


DEALT = r"""
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#include "packed_schedule.h"
using namespace fb;
#define NEED(x) do { if (!(x)) { std::printf("line %d: %s (trial %d)\n", __LINE__, #x, trial); return 1; } } while (0)

int main() {
    std::mt19937 rng(11);
    auto pick = [&](int a, int b) { return static_cast<int>(a + rng() % (b - a + 1)); };
    for (int trial = 0; trial < 2000; ++trial) {
        const int log_tokens = pick(0, 7), tokens = trial % 6 == 0 ? 0 : pick(1, trial % 3 ? 400 : 5000);
        const int before = trial % 5 == 0 ? -pick(0, tokens + 3) : trial % 2 ? 0 : pick(0, 3000);
        std::vector<int> all;
        for (int i = 0; i < tile_count(tokens, log_tokens); ++i) {
            all.push_back(key_tiles(before, tokens, log_tokens, i));
        }
        NEED(std::is_sorted(all.begin(), all.end()));
        for (int least = -1; least <= (all.empty() ? 1 : all.back()) + 2; ++least) {
            const auto those = std::count_if(all.begin(), all.end(), [&](int t) { return t >= least; });
            NEED(tiles_of_at_least(before, tokens, log_tokens, least) == those);
        }
        // Every rank is dealt to one CTA, in rounds.
        const int ctas = pick(1, 50), tiles = pick(1, 300);
        std::vector<int> dealt(tiles);
        for (int cta = 0; cta < ctas; ++cta) {
            long long before_it = -1;
            for (int round = 0; dealt_rank(round, cta, ctas) < tiles; ++round) {
                NEED(dealt_rank(round, cta, ctas) > before_it);
                before_it = dealt_rank(round, cta, ctas);
                ++dealt[before_it];
            }
        }
        NEED(std::all_of(dealt.begin(), dealt.end(), [](int n) { return n == 1; }));
    }
    const int trial = -1;
    NEED(tiles_of_at_least(0, 1 << 24, 0, 1 << 17) == 128);
    NEED(tiles_of_at_least((1 << 26) - (1 << 24), 1 << 24, 7, 1 << 19) == 1);
    return 0;
}
"""


def test_every_rank_of_whole_tiles_is_dealt_once(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "dealt.cpp").write_text(DEALT)
    subprocess.run([compiler, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(tmp_path / "dealt.cpp"), "-o", str(tmp_path / "dealt")], check=True)
    result = subprocess.run([str(tmp_path / "dealt")], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout + result.stderr
