"""Plans of experts' slots: how they lie in memory, their tiles, and what the products make of plans that are not theirs.

The header's own rules (densecore_amd/csrc/dcq_i8.h) are compiled for the CPU here, so that where a plan of another call leads is
known before any GPU reads one."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import densecore_amd as dc

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "densecore_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
LOW, HIGH = -2 ** 31, 2 ** 31 - 1

PROGRAM = r"""
#include <stdio.h>
#include <limits.h>
#include "dcq_i8.h"
using namespace dcq;
int main() {
    const int far[] = {INT_MIN, INT_MIN + 1, -65536, -2, -1, 0, 1, 2, 15, 16, 63, 64, 119, 120, 121, 127, 128, 255, 256, 4095, 4194303,
                       4194304, 4194305, INT_MAX - 256, INT_MAX - 1, INT_MAX};
    const int64_t sizes[] = {1, 2, 16, 120, 121, 4194304};
    long seen = 0;
    for (int64_t slots : sizes)
        for (int height : {16, 64, 128, 256})
            for (int n_expert : {1, 16, 512})
                for (int expert : far)
                    for (int begin : far)
                        for (int count : far) {
                            const PlanTile t = tile_inside({expert, begin, count, 0}, n_expert, slots, height);
                            ++seen;
                            const bool whole = expert >= 0 && expert <= n_expert && begin >= 0 && begin < slots && count > 0;
                            if (!whole) {
                                if (t.expert != -1) return printf("kept %d %d %d\n", expert, begin, count), 1;
                                continue;
                            }
                            if (t.expert != expert || t.begin != begin || t.count < 1 || t.count > height ||
                                (int64_t)t.begin + t.count > slots)
                                return printf("outside %d %d %d\n", expert, begin, count), 1;
                            if (count <= height && (int64_t)begin + count <= slots && t.count != count)
                                return printf("a good tile changed %d %d %d\n", expert, begin, count), 1;
                        }
    for (int64_t slots : sizes)
        for (int v : far) {
            const int s = slot_inside(v, slots);
            if (s < 0 || s >= slots || (v >= 0 && v < slots && s != v)) return printf("slot %d of %ld\n", v, (long)slots), 1;
        }
    // sizes and places: m, k, experts
    const int64_t plans[][3] = {{1, 1, 1}, {5, 8, 128}, {1000, 7, 512}, {1571, 8, 128}, {4097, 4, 60}, {3, 2, 7}, {4194304, 1, 1}, {4194304, 1, 512}};
    for (auto& p : plans) {
        const int64_t slots = p[0] * p[1];
        const int e = (int)p[2], h = plan_height(slots, e);
        printf("%ld %d %d %ld %ld %ld %ld %ld\n", (long)slots, e, h, (long)plan_order_at(e), (long)plan_expert_at(e, slots),
               (long)plan_tiles_at(e, slots), (long)plan_tiles(slots, e, h), (long)plan_ints(e, slots));
    }
    printf("%ld tiles\n", seen);
    return 0;
}
"""


def layout(slots, e):
    """(height, order's, experts' and tiles' place in int32, tiles, all) of a plan."""
    up = lambda v: -(-v // 64) * 64  # noqa: E731
    ints = dc.moe_plan_size(slots, 1, e) // 4
    order = up(e + 2)
    expert = order + up(slots)
    tiles = expert + up(slots)
    return order, expert, tiles, (ints - tiles) // 4


def test_tiles_and_slots_of_any_plan_lie_inside(tmp_path):
    if not shutil.which(HIPCC) and not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    src, exe = tmp_path / "plan.hip", tmp_path / "plan"
    src.write_text(PROGRAM)
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    lines = r.stdout.splitlines()
    assert int(lines[-1].split()[0]) == 6 * 4 * 3 * 26 ** 3
    for line in lines[:-1]:
        slots, e, height, order, expert, tiles, count, ints = map(int, line.split())
        assert layout(slots, e) == (order, expert, tiles, count) and dc.moe_plan_size(slots, 1, e) == 4 * ints
        # room for every group's last, partial tile: groups of one slot more than whole tiles
        groups, left, at = e + 1, slots, 0
        for g in range(groups):
            n = left if g == groups - 1 else min(left, max(slots // groups // height * height + 1, 1))
            t0, t1 = (at + g * (height - 1)) // height, (at + n + (g + 1) * (height - 1)) // height
            assert t1 - t0 >= -(-n // height) and t1 <= count
            left, at = left - n, at + n
        assert left == 0


# ---------------------------------------------------------------- on the GPU
def ids_of(m, e, k, seed, skew=False):
    r = np.random.default_rng(seed)
    ids = r.integers(0, e, (m, k)).astype(np.int32)
    if skew:
        ids[r.random((m, k)) < 0.7] = e // 2
    ids[r.random((m, k)) < 0.1] = -1
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("skew", [False, True])
@pytest.mark.parametrize("m,e,k,height", [(1, 1, 1, 16), (5, 128, 8, 16), (600, 512, 7, 16), (3, 7, 2, 16), (100, 4, 2, 64), (1571, 128, 8, 64),
                                          (4097, 60, 4, 128), (500, 4, 2, 128), (1100, 4, 2, 256), (9000, 3, 1, 256)])
def test_every_place_of_the_order_is_in_one_tile_of_its_expert(dev, m, e, k, height, skew):
    ids = ids_of(m, e, k, 5 * m + e, skew)
    size = dc.moe_plan_size(m, k, e)
    plan = torch.full((size,), 0x55, dtype=torch.uint8, device=dev)
    dc.moe_plan(torch.from_numpy(ids).to(dev), e, plan=plan)
    p = plan.view(torch.int32).cpu().numpy()
    slots = m * k
    order, expert, tiles, count = layout(slots, e)
    flat = np.where((ids < 0) | (ids >= e), e, ids).reshape(-1)
    of = flat[p[order:order + slots]]  # the expert of each place
    seen = np.zeros(slots, int)
    for ex, begin, n, _ in p[tiles:tiles + 4 * count].reshape(-1, 4):
        if ex == -1:
            continue
        assert 0 <= ex <= e and 0 < n <= height and 0 <= begin and begin + n <= slots
        assert (of[begin:begin + n] == ex).all()
        seen[begin:begin + n] += 1
    assert (seen == 1).all()


HEIGHTS = [(20, 16), (100, 64), (500, 128), (1100, 256), (1, 16)]  # tokens of 4 experts, 2 each; one token: one launch for down


class Call:
    """The experts' products of m tokens, with room around everything that they write."""
    e, k, n, width = 4, 2, 130, 272

    def __init__(self, dev, m):
        gen = torch.Generator(device=dev)
        gen.manual_seed(m)
        i8 = lambda *s: torch.randint(-127, 128, s, dtype=torch.int8, device=dev, generator=gen)  # noqa: E731
        f32 = lambda *s: 0.002 + 0.01 * torch.rand(s, device=dev, generator=gen)  # noqa: E731
        self.m, self.slots = m, m * self.k
        self.ids = torch.from_numpy(ids_of(m, self.e, self.k, m)).to(dev)
        if m == 1:
            self.ids[:] = torch.tensor([[1, 3]], dtype=torch.int32)
        self.up_args = (i8(self.e, self.n, self.width), f32(self.e, self.n), i8(self.e, self.n, self.width), f32(self.e, self.n),
                        i8(m, self.width), f32(m), self.k)
        self.down_args = (i8(self.e, self.n, self.width), f32(self.e, self.n), i8(self.slots, self.width), f32(self.slots), f32(m, self.k))
        self.plan = dc.moe_plan(self.ids, self.e)
        self.size = dc.moe_down_i8_workspace_size(m, self.k, self.n)
        self.h = torch.empty((self.slots + 64, self.n), device=dev)
        self.y = torch.empty((m + 64, self.n), device=dev)
        self.ws = torch.empty(self.size + 2 * 65536, dtype=torch.uint8, device=dev)
        self.want = [t.clone() for t in self.run(self.plan)]

    def run(self, plan):
        """(H, Y), where all that lies around them has to be left as it was."""
        self.h.fill_(7)
        self.y.fill_(7)
        self.ws.fill_(0x55)
        h, y = self.h[32:32 + self.slots], self.y[32:32 + self.m]
        dc.moe_gate_up_i8(plan, *self.up_args, h=h)
        dc.moe_down_i8(plan, *self.down_args, y=y, workspace=self.ws[65536:65536 + self.size])
        torch.cuda.synchronize()
        for t, rows in ((self.h, self.slots), (self.y, self.m)):
            assert (t[:32] == 7).all() and (t[32 + rows:] == 7).all()
        assert (self.ws[:65536] == 0x55).all() and (self.ws[65536 + self.size:] == 0x55).all()
        return h, y

    def sections(self):
        """A copy of the plan, and its order, experts and tiles as views of it."""
        p = self.plan.clone()
        v = p.view(torch.int32)
        order, expert, tiles, count = layout(self.slots, self.e)
        return p, v[order:order + self.slots], v[expert:expert + self.slots], v[tiles:tiles + 4 * count].view(-1, 4)


def far(n, dev, *values):
    return torch.tensor(values, dtype=torch.int64, device=dev).repeat(-(-n // len(values)))[:n].int()


@pytest.mark.gpu
@pytest.mark.parametrize("m,height", HEIGHTS)
def test_slots_past_the_arrays_under_valid_tiles(dev, m, height):
    c = Call(dev, m)
    for values in ((-1,), (LOW, HIGH), (c.slots, c.slots + 1, -c.slots), (0, -1, c.slots - 1, 1 << 22)):
        p, order, _, _ = c.sections()
        order.copy_(far(c.slots, dev, *values))
        c.run(p)
    # every other place: rows that the remaining ones name are theirs all the same, but for the last, where those outside go
    p, order, _, _ = c.sections()
    kept = order.clone()
    order[::2] = far(len(order[::2]), dev, LOW, -1, c.slots, HIGH)
    h, _ = c.run(p)
    rows = kept[1::2].long()
    rows = rows[rows != c.slots - 1]
    assert torch.equal(h[rows], c.want[0][rows])


@pytest.mark.gpu
@pytest.mark.parametrize("m,height", HEIGHTS)
def test_tiles_past_the_arrays(dev, m, height):
    c = Call(dev, m)
    used = [i for i, t in enumerate(c.sections()[3].tolist()) if t[0] >= 0]
    for column, values in ((0, (c.e + 1, HIGH)), (0, (LOW, -2)), (0, (c.e,)), (1, (c.slots, HIGH)), (1, (-1, LOW)), (1, (c.slots - 1,)),
                           (1, (max(c.slots - 5, 0),)), (2, (HIGH, height + 1)), (2, (0, -1, LOW))):
        p, _, _, tiles = c.sections()
        tiles[:, column] = far(len(tiles), dev, *values)
        c.run(p)
    # unused tiles that claim rows, and all of the section past the arrays
    p, _, _, tiles = c.sections()
    tiles[tiles[:, 0] < 0] = torch.tensor([c.e - 1, c.slots - 1, HIGH, 0], dtype=torch.int32, device=dev)
    c.run(p)
    for value in (LOW, HIGH, c.slots - 1, c.e):
        p, _, _, tiles = c.sections()
        tiles.fill_(value)
        c.run(p)
    # a tile whose expert, begin or count is out of range is left out; the others' rows are as they were
    for column, value in ((0, c.e + 1), (0, -3), (1, c.slots), (1, LOW), (2, 0), (2, -7)):
        p, order, _, tiles = c.sections()
        at = used[len(used) // 2]
        _, begin, n, _ = tiles[at].tolist()
        tiles[at, column] = value
        h, _ = c.run(p)
        rows = order[begin:begin + n].long()
        want = c.want[0].clone()
        want[rows] = 7
        assert torch.equal(h, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,height", HEIGHTS)
def test_experts_of_slots_past_the_arrays(dev, m, height):
    """The part that the sums of a token and the one-token launch read."""
    c = Call(dev, m)
    for values in ((LOW, -2), (c.e,), (c.e + 1, HIGH), (-1,)):
        p, _, expert, _ = c.sections()
        expert.copy_(far(c.slots, dev, *values))
        h, y = c.run(p)
        assert torch.equal(h, c.want[0])
        if values[0] < 0:
            assert (y == 0).all()
    p, _, _, _ = c.sections()
    p.view(torch.int32)[:c.e + 2] = far(c.e + 2, dev, HIGH, LOW)  # offsets: the products do not read them
    h, y = c.run(p)
    assert torch.equal(h, c.want[0]) and torch.equal(y, c.want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("m,height", HEIGHTS)
def test_a_plan_of_other_sizes_stays_inside(dev, m, height):
    """A real plan of other tokens and experts."""
    c = Call(dev, m)
    for other, e, k in ((3 * m + 7, 9, 2), (max(m // 2, 1), 3, 4), (m, 512, 2), (40 * m, 2, 1)):
        ids = torch.from_numpy(ids_of(other, e, k, other)).to(dev)
        bytes_ = dc.moe_plan(ids, e)
        p = torch.full_like(c.plan, 0x55)
        n = min(len(p), len(bytes_))
        p[:n] = bytes_[:n]
        c.run(p)
