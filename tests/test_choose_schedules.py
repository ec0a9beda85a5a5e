"""The choice of the best pages (csrc/pfa_choose.h) followed on the CPU, with the
waves of its workgroup in chosen orders: what a wave leaves in LDS must not reach
another wave before a barrier says so, whatever wave is ahead."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "proteus-flux-attention_amd" / "csrc"
NONE, NAN, FORCED = 0, 1, 0xffffffff

# threads and entries of each form; the last takes rows of any length, in rounds
FORMS = [(256, 512), (256, 1024), (1024, 4096), (1024, 8192), (1024, 16384), (1024, 40000)]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("choose")
    lines = (CSRC / "pfa_choose.h").read_text().splitlines()
    (tmp / "choose.h").write_text("\n".join(x for x in lines if not x.startswith("#include")) + "\n")
    lib = tmp / "libchoose.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w", f"-I{tmp}", str(HERE / "choose_on_host.cpp"),
                    "-o", str(lib)], check=True)
    fn = ctypes.CDLL(str(lib)).choose_on_host
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731

    def call(form, keys, count, order):
        keys, order = np.ascontiguousarray(keys, np.uint32), np.ascontiguousarray(order, np.int32)
        out = np.full(count, -7, np.int32)
        assert fn(form, ptr(keys), len(keys), count, ptr(order), ptr(out)) == 0, "waves that do not meet"
        return out

    return call


def _best(keys, count):
    """The definition: forced and large keys first, ties by entry; ascending, -1 behind."""
    held = np.flatnonzero(keys != NONE)
    take = np.sort(held[np.lexsort((held, -keys[held].astype(np.int64)))][:count])
    return np.concatenate([take, np.full(count - len(take), -1)]).astype(np.int32)


def _orders(waves, rng):
    up = np.arange(waves)
    yield up
    yield up[::-1].copy()
    yield np.roll(up, 1)
    yield rng.permutation(waves)


def _rows(n, rng):
    """Keys of a row, by what decides the choice."""
    some = rng.integers(2, 0xff800001, n, dtype=np.uint32)
    some[rng.random(n) < 0.1] = NONE
    ends = some.copy()
    ends[:2] = ends[-3:] = FORCED
    gone = np.full(n, NONE, np.uint32)
    gone[rng.integers(0, n, 5)] = FORCED
    yield "all taken, forced ones among them", ends, n + 3
    yield "all taken, none forced", some, n
    yield "only forced ones", ends, 5
    yield "forced ones and holes", gone, 9
    yield "all alike", np.full(n, 0x80000000, np.uint32), n // 3 + 1
    yield "all alike behind forced ones", np.where(ends == FORCED, FORCED, 0x80000000).astype(np.uint32), n // 2
    yield "cut once", (ends & ~np.uint32(0x3ff)) | (ends == FORCED) * np.uint32(FORCED), n // 4 + 5
    yield "cut to the last bit", np.where(ends == FORCED, ends, 0x80000000 + ends % 7).astype(np.uint32), n // 2
    yield "not a number", np.where(some == NONE, NONE, NAN).astype(np.uint32), n // 2
    yield "nothing", np.full(n, NONE, np.uint32), 4
    # more to take than a wave's count of what it takes can be mistaken for
    yield "more than there are by far", ends, (1 << 16) + n


@pytest.mark.parametrize("form", range(len(FORMS)), ids=lambda f: f"{FORMS[f][0]}x{FORMS[f][1]}")
def test_any_wave_ahead(choose, form):
    threads, most = FORMS[form]
    rng = np.random.default_rng(form)
    for n in (most, most - 3, most // 2 + 1):
        for what, keys, count in _rows(n, rng):
            want = _best(keys, count)
            for order in _orders(threads // 64, rng):
                got = choose(form, keys, count, order)
                assert np.array_equal(got, want), (what, n, count, order.tolist(), int((got != want).sum()))
