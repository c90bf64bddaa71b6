"""The decoders' sequence cache (csrc/host_cache.h), compiled by itself: places that are taken back leave it as it was."""
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "koboldcpp_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "host_cache.h"
using b200::host::SeqCache;

static bool same(const SeqCache &a, const SeqCache &b) {
    if (a.cell_seq != b.cell_seq || a.cell_pos != b.cell_pos || a.n_used != b.n_used || a.high != b.high || a.seqs.size() != b.seqs.size()) return false;
    for (size_t i = 0; i < a.seqs.size(); i++)
        if (a.seqs[i].open != b.seqs[i].open || a.seqs[i].fresh != b.seqs[i].fresh || a.seqs[i].lost != b.seqs[i].lost || a.seqs[i].len != b.seqs[i].len) return false;
    return true;
}
// no free cell below first_free
static bool sound(const SeqCache &c) {
    for (int i = 0; i < c.first_free && i < c.n_cells(); i++) if (c.cell_seq[(size_t)i] < 0) return false;
    return true;
}

int main() {
    srand(1);
    for (int run = 0; run < 300; run++) {
        SeqCache c;
        c.init(40, 5);
        for (int step = 0; step < 60; step++) {
            const int what = rand() % 4;
            if (what == 0) c.open_seq();
            if (what == 1) c.close_seq(rand() % 5);
            if (what < 2) continue;
            // a step over the open sequences; half of them are taken back
            const SeqCache before = c;
            std::vector<int> ids, counts;
            std::vector<std::vector<int32_t>> cells;
            for (int id = 0; id < 5; id++) {
                const int n = rand() % 6;
                std::vector<int32_t> at((size_t)n + 1), pos((size_t)n + 1);
                if (!c.place(id, n, at.data(), pos.data())) continue;
                for (int i = 0; i < n; i++) if (pos[(size_t)i] != before.seqs[(size_t)id].len + i) { printf("positions\n"); return 1; }
                ids.push_back(id); counts.push_back(n); cells.push_back(at);
            }
            if (!sound(c)) { printf("placed\n"); return 1; }
            if (what == 3) continue;
            for (size_t i = 0; i < ids.size(); i++) c.unplace(ids[i], counts[i], cells[i].data());
            if (!same(before, c) || !sound(c)) { printf("run %d step %d: not as it was\n", run, step); return 1; }
        }
    }
    SeqCache c;
    c.init(8, 2);
    c.seqs[(size_t)c.open_seq()].lost = true;
    c.close_seq(0);
    return c.seqs[(size_t)c.open_seq()].lost ? 1 : 0;
}
"""


def test_places_that_are_taken_back(tmp_path):
    src = tmp_path / "cache.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", str(CSRC), str(src), "-o", str(tmp_path / "cache")], check=True)
    r = subprocess.run([str(tmp_path / "cache")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
