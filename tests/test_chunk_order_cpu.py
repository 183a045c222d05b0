"""The order in which chunk attention's ring is filled and waited for, gone through on the host."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIMS = (32, 64, 96, 128, 192, 256)
MOST = 24  # steps of a segment: more than twice a ring

PROGRAM = """
#include <cstdio>
#include <initializer_list>
#include "hv_chunk_order.cuh"
using namespace hv::chunk;
static_assert(!order_of(256).values_may_be_polled(false, 12) && order_of(256).values_may_be_polled(true, 12), "at compile time too");
int main() {
    for (int d : {32, 64, 96, 128, 192, 256}) {
        const Order o = order_of(d);
        printf("%d %d %d %d %d %d\\n", o.apart, o.parts, o.stages, o.row_tiles, o.values_may_be_polled(false, 24), o.values_may_be_polled(true, 24));
        for (int lead = 1; lead <= 2; ++lead)
            for (int n = 1; n <= 24; ++n)
                for (int j = 0; j < n; ++j) printf("%d %d ", o.k_fill(j, lead), o.v_fill(j, n, lead));
        printf("\\n");
    }
}
"""


@pytest.fixture(scope="module")
def orders(tmp_path_factory):
    d = tmp_path_factory.mktemp("order")
    (d / "order.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "heatvit_b200", "csrc"), str(d / "order.cpp"), "-o",
                    str(d / "order")], check=True)
    lines = iter(subprocess.run([str(d / "order")], capture_output=True, text=True, check=True).stdout.splitlines())
    out = {}
    for dim in DIMS:
        apart, parts, stages, tiles, early, late = map(int, next(lines).split())
        numbers = iter(map(int, next(lines).split()))
        fills = {(lead, n): [(next(numbers), next(numbers)) for _ in range(n)] for lead in (1, 2) for n in range(1, MOST + 1)}
        out[dim] = (apart, parts, stages, tiles, early, late, fills)
    return out


def copies(n, lead, apart):
    """What the copying warps fill, one after the other."""
    order = [("k", j) for j in range(min(lead, n))]
    for j in range(n):
        if not apart:
            order.append(("v", j))
        if j + lead < n:
            order.append(("k", j + lead))
        if apart:
            order.append(("v", j))
    return order


def products(units, tiles, apart):
    """What the products' warp waits for, one after the other."""
    order = []
    for i in range(units + tiles):
        for first in (True, False):
            if first == bool(apart):
                order += [("k", i)] if i < units else []
            else:
                order += [("v", i - tiles)] if i >= tiles else []
    return order


@pytest.mark.parametrize("dim", DIMS)
def test_fills_are_counted_as_they_are_copied(orders, dim):
    apart, parts, _, tiles, _, _, fills = orders[dim]
    for lead in range(1, tiles + 1):
        for n in range(1, MOST + 1):
            for i, (kind, j) in enumerate(copies(n, lead, apart)):
                assert fills[lead, n][j]["kv".index(kind)] == i * parts


@pytest.mark.parametrize("dim", DIMS)
def test_a_polled_slot_is_past_its_earlier_fill(orders, dim):
    """A parity tells a fill from the one ahead of it alone, so whoever polls a slot's barrier must know the earlier fill
    landed.  A softmax warpgroup that looks through a step's values knows what the products' warp waited for ahead of the
    scores of its unit, and of the sums of its unit before where it awaits those."""
    apart, parts, stages, tiles, early, late, _ = orders[dim]

    def sound(sums_ahead):
        for alt in range(tiles):
            pair = tiles == 2 and not alt
            per = 2 if pair else 1
            for n in range(1, MOST + 1):
                owner = [c for c in copies(n, 2 if alt else 1, apart) for _ in range(parts)]
                order = products(n * per, tiles, apart)
                for u in range(n * per):
                    known = order.index(("k", u))
                    if sums_ahead and u >= tiles:
                        known = max(known, order.index(("v", u - tiles)))
                    waited = {(kind, unit // per) for kind, unit in order[:known + 1]}
                    at = owner.index(("v", u // per))
                    if any(f - stages >= 0 and owner[f - stages] not in waited for f in range(at, at + parts)):
                        return False
        return True
    assert sound(True) and late
    assert sound(False) == bool(early) == (dim != 256)
