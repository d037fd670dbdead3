"""The packed prefill's list of runs on the CPU: csrc/paged_plan.h built for the host
(paged_plan_host.cpp), its lists against what the lengths say.  Every unit of every tile
of every KV head in exactly one run, every index inside what it names, every part of a
cut tile at its place, nothing written outside the workspace's entries."""
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROWS, UNIT, LIST = 128, 32, 1024
RUN = ("tile", "u0", "u1", "part", "cu", "nq", "past", "z", "tok", "head")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "plan")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wno-unknown-pragmas", "-I", os.path.join(HERE, "..", "include"),
                    os.path.join(HERE, "paged_plan_host.cpp"), "-o", exe], check=True)
    return exe


class Words:
    def __init__(self, raw):
        self.w, self.at = np.frombuffer(raw, np.int32), 0

    def take(self, n):
        self.at += n
        return self.w[self.at - n:self.at].tolist()

    def entries(self, size):
        out = {}
        while (i := self.take(1)[0]) >= 0:
            assert i not in out
            out[i] = self.take(size)
        return out


def ceil(a, b):
    return -(-a // b)


def check(call, words):
    """One call's output: (tiles, whether tiles could be cut, cut tiles) of each launch."""
    launches = words.take(1)[0]
    out, at = [], 0
    for _ in range(launches):
        begin, end, *sizes = words.take(7)
        assert begin == at < end
        at = end
        out.append(check_launch(call, begin, end, sizes, words))
    assert at == call["head"][1]
    return out


def check_launch(call, begin, end, sizes, words):
    cus, n, B, G, hkv, log, W = call["head"]
    length = call["len"]
    cu = np.clip(call["cu"], begin, end).tolist()
    most, slots, wgs, n_runs, n_cuts = sizes
    total, cuts, kind = words.take(3)
    assert most <= LIST and n_runs <= LIST and total <= LIST
    runs, cut = words.entries(12), words.entries(8)
    cap = W << log
    tiles = {}
    for z in range(B):
        nq = cu[z + 1] - cu[z]
        past = min(max(length[z], 0), cap) - (call["cu"][z + 1] - cu[z])
        for t in range(ceil(nq * G, ROWS)):
            last = min((t + 1) * ROWS, nq * G) - 1
            tiles[z, t] = ceil(max(past + last // G + 1, 0), UNIT), nq, past
    assert len(tiles) <= most
    assert total * hkv <= wgs and 0 <= total
    assert all(0 <= i < n_cuts for i in cut)
    if kind == 0:                                   # a record for all heads, in any order
        assert sorted(runs) == list(range(total)) and total <= n_runs
        found = [(r, h) for r in runs.values() for h in range(hkv)]
        assert len(tiles) > slots
    else:                                           # a record a workgroup
        found = [(r, r[9]) for r in runs.values() if r[9] >= 0]
        assert len(found) == total * hkv and total <= slots
        if kind == 1:
            assert sorted(runs) == list(range(ceil(total * hkv, 8) * 8)) and len(runs) <= min(n_runs, wgs)
    by = {}
    for r, h in found:
        r = dict(zip(RUN, r))
        assert 0 <= h < hkv and (r["z"], r["tile"]) in tiles, r
        units, nq, past = tiles[r["z"], r["tile"]]
        assert (r["cu"], r["nq"], r["past"], r["tok"]) == (cu[r["z"]], nq, past, r["tile"] * ROWS // G), r
        by.setdefault((r["z"], r["tile"], h), []).append(r)
    assert len(by) == len(tiles) * hkv
    joins = {(c[0], c[3], c[4]): c for c in cut.values()}
    assert len(joins) == len(cut)
    used = []
    for (z, t, h), rs in by.items():
        units, nq, _ = tiles[z, t]
        rs.sort(key=lambda r: r["u0"])
        assert rs[0]["u0"] == 0 and rs[-1]["u1"] == units
        assert all(a["u1"] == b["u0"] for a, b in zip(rs, rs[1:]))
        assert len(rs) == 1 or all(r["u0"] < r["u1"] for r in rs)
        c = joins.get((t, cu[z], nq))
        if len(rs) == 1:
            assert rs[0]["part"] == -1 and (kind == 2 or c is None)
            assert c is None or c[2] == 1
        else:
            assert c is not None and c[2] == len(rs)
            assert [r["part"] for r in rs] == list(range(c[1], c[1] + c[2])) and c[1] + c[2] <= slots
            if h == 0:
                used += range(c[1], c[1] + c[2])
    assert len(set(used)) == len(used)
    many = sum(len(rs) > 1 for (_, _, h), rs in by.items() if h == 0)
    assert sorted(cut) == list(range(cuts)) and cuts == (len(tiles) if kind == 2 else many)
    return len(tiles), kind, many


def make(new, past, G, hkv, page=64, cus=256, table=None, begin=0, behind=0):
    length = [a + b for a, b in zip(new, past)]
    cu = (begin + np.concatenate([[0], np.cumsum(new)])).tolist()
    W = table or max(1, ceil(max(length), page))
    return {"head": (cus, cu[-1] + behind, len(new), G, hkv, page.bit_length() - 1, W), "cu": cu, "len": length}


def run(program, calls, rcp=0, descending=0):
    text = "\n".join(" ".join(map(str, [*c["head"], *c["cu"], *c["len"]])) for c in calls)
    out = subprocess.run([program, str(rcp), str(descending)], input=text.encode(), stdout=subprocess.PIPE, check=True)
    words = Words(out.stdout)
    result = [check(c, words) for c in calls]
    assert words.at == len(words.w)
    return result


CALLS = {
    "one token": make([1], [0], 4, 5),
    "a first turn": make([101], [0], 4, 5),
    "drafts": make([1, 5, 2, 4] * 6, [4000, 600, 1200, 3000] * 6, 4, 5),
    "idle sequences": make([33, 0, 1, 64, 0], [0, 50, 300, 5, 0], 4, 5, begin=3, behind=20),
    "more sequences than lanes": make([3, 0, 40] * 40, [7, 100, 900] * 40, 2, 3),
    "as many as a call takes": make([1] * 128, list(range(128)), 1, 1),
    "a prompt that is cut": make([2048], [0], 4, 5),
    "a turn behind a long cache": make([333, 40, 12], [30011, 3000, 90], 4, 5, page=128),
    "more KV heads than workgroups": make([3, 9], [40, 60], 1, 600),
    "whole rounds": make([2048] * 4, [0] * 4, 4, 5),
    "tiles past a round": make([3300], [20000], 4, 5),
    "tiles past a round of small groups": make([1030], [2500], 8, 8),
    "packed prompts": make([4096, 1700, 900, 0, 2300, 600], [0] * 6, 4, 5),
    "a group of more heads than rows": make([3, 0, 9], [40, 5, 60], 200, 1),
    "nothing to see": make([40, 6, 10], [-37, -6, -9], 2, 2),
    "few CUs": make([900, 70], [100, 3000], 4, 2, cus=3),
    "1016 tiles": make([4064] * 8, [0] * 8, 4, 5),
}


@pytest.mark.parametrize("descending", [0, 1])
@pytest.mark.parametrize("rcp", [-1, 0, 1])
def test_calls(program, rcp, descending):
    for (name, call), [(tiles, kind, cut)] in zip(CALLS.items(), run(program, CALLS.values(), rcp, descending)):
        if name in ("one token", "a first turn", "drafts"):
            assert kind == 2, name                  # no list
        if name in ("whole rounds", "packed prompts", "1016 tiles"):
            assert kind == 0 and not cut, name
        if "past a round" in name:
            assert kind == 0 and cut, name
    assert tiles == 1016


def test_calls_at_random(program):
    rng = np.random.default_rng(11)
    calls = []
    for _ in range(60):
        B = int(rng.choice([1, 2, 5, 30, 64, 65, 128]))
        hkv, G = int(rng.choice([1, 2, 5, 8, 33])), int(rng.choice([1, 2, 3, 4, 7, 8, 16]))
        most = int(2 ** rng.uniform(0, 12)) // B + 1
        new = rng.integers(0, min(most, 900 * ROWS // (G * B)) + 1, B).tolist()
        new[0] += not sum(new)
        past = (rng.integers(0, int(2 ** rng.uniform(0, 14)) + 1, B) * rng.integers(0, 2, B)).tolist()
        calls.append(make(new, past, G, hkv, int(rng.choice([32, 64, 256])), int(rng.choice([256, 256, 64])),
                          begin=int(rng.integers(0, 3)), behind=int(rng.integers(0, 40))))
    kinds = [k for r in run(program, calls) for _, k, _ in r]
    assert {0, 1, 2} == set(kinds)


LONG = {
    "1025 tiles": make([32800], [0], 4, 5),
    "1025 tiles of 16 heads": make([8200], [700], 16, 2),
    "prompts of many launches": make([30000, 0, 70001, 1, 4000], [0, 9, 100, 5, 20000], 4, 5),
    "a whole batch": make([1000, 1, 90] * 42, [0, 3000, 40] * 42, 6, 2, begin=5, behind=300),
    "one KV head": make([140000], [2000], 1, 1, page=256),
    "four times the list": make([32] * 128, list(range(128)), 128, 1),
    "a token is 512 tiles": make([3, 2], [50, 900], 65535, 1),
    "few CUs": make([9000, 300], [0, 70], 16, 3, cus=7),
    "behind the last token": make([40], [0], 4, 5, behind=40000),
}


@pytest.mark.parametrize("descending", [0, 1])
def test_long_lists_go_in_several(program, descending):
    """More tiles than a list takes: launches that follow one another, each a list of
    1024 at most, every token in one of them."""
    for (name, call), out in zip(LONG.items(), run(program, LONG.values(), 0, descending)):
        most = call["head"][1] * call["head"][3] // ROWS + len(call["len"])
        assert 1 < len(out) <= 2 * most // LIST + 2, name
        assert sum(t for t, _, _ in out) >= sum(ceil(a * call["head"][3], ROWS) for a in np.diff(call["cu"])), name
