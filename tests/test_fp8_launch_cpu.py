"""CPU: which kernel the 8-bit products launch, and how they cut it over
clusters, for a device that a fake CUDA runtime (fake_cuda_runtime.c) stands
for.  Each sequence of calls runs in a process of its own, with the fake
preloaded; addresses are made up, nothing is read or launched."""
import ctypes
import importlib.util
import json
import os
import re
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

HERE = os.path.dirname(os.path.abspath(__file__))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
pytestmark = pytest.mark.skipif(shutil.which("gcc") is None or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime_api.h")),
                                reason="gcc or the CUDA headers not available")


def child(calls):
    """In a process with the fake preloaded: [status, launches] of each call (tokens, rows, k, parts, the output's type of a
    product of one part, whether the handle was initialised)."""
    spec = importlib.util.spec_from_file_location("zkv_lib", os.path.join(ROOT, "zoomkv_revision_b200", "_lib.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    lib, fake = mod.lib(), ctypes.CDLL(None)
    fake.fake_launches.restype = ctypes.c_char_p
    got = []
    for tokens, rows, k, parts, kind, init in calls:
        w = mod.ZkvFp8Weight(w=1 << 32, scale=1 << 33, ld=k, rows=rows, k=k, parts=parts)
        assert not init or lib.zkv_fp8_weight_init(ctypes.addressof(w)) == 0
        fake.fake_forget()
        x = (1 << 34, k, 1 << 35, 1, max(tokens, 1), tokens, ctypes.addressof(w), 1 << 36, rows)
        rc = lib.zkv_fp8_linear(*x, kind, None, None) if parts == 1 else lib.zkv_fp8_swiglu(*x, 1 << 37, 1, max(tokens, 1), None, None)
        got.append([rc, fake.fake_launches().decode()])
    return got


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    so = tmp_path_factory.mktemp("fake") / "fake.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-Wall", "-I", os.path.join(CUDA, "include"), "-o", str(so),
                    os.path.join(HERE, "fake_cuda_runtime.c")], check=True)

    def run(calls, how="one"):
        calls = [(*c, *(0, True)[len(c) - 4:]) for c in calls]
        env = dict(os.environ, LD_PRELOAD=str(so), FAKE_CTAS_AN_SM=how)
        out = subprocess.run([sys.executable, os.path.abspath(__file__), json.dumps(calls)], env=env, capture_output=True,
                             text=True, timeout=60)
        assert out.returncode == 0, out.stderr[-2000:]
        got = []
        for rc, text in json.loads(out.stdout.splitlines()[-1]):
            lines = []
            for line in text.splitlines():
                name, x, y, cluster = line.split()
                few = re.search(r"few_kernelILi(\d+)ELi(\d)E", name)
                many = re.search(r"many_kernelILb([01])E", name)
                lines.append((f"few {few[1]} {few[2]}" if few else f"many {int(many[1]) + 1}", int(x), int(y), int(cluster)))
            got.append((rc, lines))
        return got
    return run


# tokens, rows, k, parts: a decode step's products, few and many tokens, each kernel at least once
SHAPES = [(1, 6144, 4096, 1), (8, 4096, 4096, 1), (8, 4096, 12288, 1), (32, 4096, 12288, 1), (32, 151936, 4096, 1),
          (64, 4096, 4096, 1), (100, 6144, 4096, 1), (333, 4096, 4096, 1), (512, 4096, 12288, 1), (768, 4096, 4096, 1),
          (4096, 6144, 4096, 1), (8, 12288, 4096, 2), (32, 12288, 4096, 2), (64, 2048, 4096, 2), (100, 12288, 4096, 2),
          (129, 12288, 4096, 2), (300, 1024, 4096, 2), (8191, 12288, 4096, 2)]


def test_a_call_is_cut_the_same_whichever_came_before(launches):
    """Nor does it matter whether the occupancy call counts the CTAs that an SM holds or one."""
    want = launches(SHAPES)
    assert all(rc == 0 and len(lines) == 1 for rc, lines in want)
    assert {lines[0][0] for _, lines in want} == {"few 16 1", "few 32 1", "few 64 1", "few 128 1", "few 16 2", "few 32 2",
                                                  "few 64 2", "few 128 2", "many 1", "many 2"}
    for how in ("one", "footprint"):
        for first in (SHAPES[0], SHAPES[3], SHAPES[6], SHAPES[10], SHAPES[11], SHAPES[14]):
            assert launches([first] + SHAPES, how)[1:] == want, (how, first)


def test_two_ctas_share_an_sm(launches):
    """Up to 32 tokens: 32 tiles of 96 blocks fit the device at once in clusters of eight, 48 of 32 blocks in clusters of four,
    where two CTAs share an SM, whatever the occupancy calls count.  64 tokens have an SM a CTA."""
    for how in ("one", "footprint"):
        got = launches([(8, 4096, 12288, 1), (32, 4096, 12288, 1), (1, 6144, 4096, 1), (64, 4096, 12288, 1)], how)
        assert got == [(0, [("few 16 1", 256, 1, 8)]), (0, [("few 32 1", 256, 1, 8)]), (0, [("few 16 1", 192, 1, 4)]),
                       (0, [("few 64 1", 128, 1, 4)])]


def test_millions_of_tokens(launches):
    """A grid has room for 65535 tiles of tokens; the pairs take more."""
    most = 65535 * 128
    got = launches([(most, 128, 8192, 1), (most + 1, 128, 8192, 1), (2 * most, 16, 6528, 1), (most + 1, 128, 8192, 2)])
    assert [rc for rc, _ in got] == [0] * 4
    assert [lines[0][0] for _, lines in got] == ["few 128 1", "many 1", "many 1", "many 2"]
    assert got[0][1][0][2] == 65535


def test_the_pairs_sizes(launches):
    """Sizes that the GPU tests mean for the pairs are theirs, whatever the output's type; and one tile of tokens more."""
    sizes = [(2048, 4096, 1024), (1500, 4001, 1040), (1600, 4096, 1040), (2049, 4001, 1040)]
    for rc, lines in launches([(*x, 1, kind) for x in sizes for kind in (0, 1, 3)]):
        assert rc == 0 and [name for name, *_ in lines] == ["many 1"]


def test_a_handle_that_was_not_initialised_is_refused(launches):
    """Its tensor map would be read by the copies as it is; a call of no tokens reads none."""
    for tokens, parts in [(1, 1), (100, 1), (4096, 1), (8, 2), (4096, 2)]:
        assert launches([(tokens, 4096, 1024, parts, 0, False)]) == [(1, [])]
    assert launches([(0, 4096, 1024, parts, 0, False) for parts in (1, 2)]) == [(0, [])] * 2


if __name__ == "__main__":
    print(json.dumps(child(json.loads(sys.argv[1]))))
