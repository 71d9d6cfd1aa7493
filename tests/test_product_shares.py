"""How the wide form of the catalogue loss shares out its matrix products (csrc/xent_plan.h), walked on the CPU: every tile is the sum of
exactly its own parts, and no part is written over another."""
import os
import random
import shutil
import subprocess

import pytest

from conftest import ROOT

WALK = r'''
#include <cstdio>
#include <cstdlib>
#include <map>
#include <vector>
#include "xent_plan.h"
using namespace xent;
#define REQUIRE(c) do { if (!(c)) { std::printf("%s: size %d, %lld x %lld x %lld\n", #c, size, (long long)M, (long long)N, (long long)K); return 1; } } while (0)

int main(int argc, char** argv)
{
    long long own = 0, shared = 0;
    for (int a = 1; a + 3 < argc; a += 4) {
        const int size = std::atoi(argv[a]);
        const int64_t M = std::atoll(argv[a + 1]), N = std::atoll(argv[a + 2]), K = std::atoll(argv[a + 3]);
        const ProductPlan p = product_plan(size, M, N, K);
        REQUIRE(p.tiles_m * p.tile >= M && p.tiles_n * p.tile >= N && p.steps * TB >= K && p.share * p.workers >= p.units && p.workers <= places_of(p.tile));
        struct Place { int64_t tile, count; };
        std::map<int64_t, Place> places;                               // what each place holds at the end of the launch
        std::vector<int64_t> finished(p.tiles_m * p.tiles_n), steps(p.tiles_m * p.tiles_n);
        for (int64_t w = 0; w < p.workers; ++w) {
            const int64_t end = (w + 1) * p.share < p.units ? (w + 1) * p.share : p.units;
            REQUIRE(w * p.share < end);
            for (int64_t u = w * p.share; u < end;) {
                const TilePart q = tile_part(u, end, p.steps);
                REQUIRE(q.count > 0 && q.step + q.count <= p.steps);
                u += q.count;
                steps[q.tile] += q.count;
                if (q.count == p.steps) { finished[q.tile]++; own++; continue; }
                const int64_t place = place_of_part(w, q.step == 0);
                REQUIRE(places.count(place) == 0);                      // nothing lies there yet
                REQUIRE((size_t)(place + 1) * p.tile * p.tile <= p.floats);
                places[place] = Place{q.tile, q.count};
                shared++;
            }
        }
        for (int64_t t = 0; t < p.tiles_m * p.tiles_n; ++t) {
            REQUIRE(steps[t] == p.steps);
            const Workers from = workers_of(t, p.steps, p.share);
            REQUIRE(finished[t] == (from.first == from.last));
            if (finished[t]) continue;
            int64_t joined = 0;
            for (int64_t w = from.first; w <= from.last; ++w) {
                const auto at = places.find(place_of_part(w, w == from.first));
                REQUIRE(at != places.end() && at->second.tile == t);
                joined += at->second.count;
            }
            REQUIRE(joined == p.steps);
            REQUIRE(p.share % p.steps != 0);                            // else join_kernel is not launched
        }
    }
    std::printf("ok %lld %lld\n", own, shared);
    return 0;
}
'''

# element size, M, N, K of dx (tokens, width, piece) and of dw (piece, width, tokens)
LISTED = [(2, 8192, 4096, 8192), (2, 8192, 4096, 808), (2, 16384, 2048, 4096), (2, 4224, 4096, 15872), (2, 32768, 768, 2048), (2, 16385, 1024, 3840),
          (4, 16384, 600, 2048), (4, 8192, 1280, 4096), (4, 8193, 1000, 260), (2, 4096, 1024, 16384), (2, 16384, 1024, 4096), (4, 3706, 500, 6040), (4, 1, 700, 1),
          (4, 600, 384, 7296), (2, 129, 129, 128), (2, 128, 4096, 131072)]


def test_every_tile_is_joined_from_its_own_parts(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(WALK)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "recommender_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    rng = random.Random(7)
    sizes = list(LISTED)
    for _ in range(3000):
        m, n, k = (int(2 ** rng.uniform(0, top)) for top in (15.5, 13, 15))
        sizes.append((rng.choice((2, 4)), m, n, k) if rng.random() < 0.5 else (rng.choice((2, 4)), k, n, m))
    own = shared = 0
    for at in range(0, len(sizes), 500):
        out = subprocess.run([str(exe)] + [str(v) for s in sizes[at:at + 500] for v in s], capture_output=True, text=True)
        assert out.returncode == 0, out.stdout
        own, shared = own + int(out.stdout.split()[1]), shared + int(out.stdout.split()[2])
    assert own > 10000 and shared > 10000                                # both kinds were walked
