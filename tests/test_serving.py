"""Block tables on the GPU, pages in 4 bits and log probabilities: what is refused before anything is launched, and the
plain implementations against one another (no GPU needed)."""

from __future__ import annotations

import ctypes
import random
import threading
from pathlib import Path

import pytest
import torch
from plain import serving_plain as plain

from lockstep_amd.ops import Fp4Pages, KernelError, kernels
from lockstep_amd.ops import build as kernel_build


def test_nearest_levels():
    x = torch.zeros(64)
    x[:9] = torch.tensor([6.0, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -5.0, 5.1])
    want = torch.zeros(64, dtype=torch.float64)
    want[:9] = torch.tensor([6.0, 0.0, 1.0, 1.0, -2.0, 2.0, 4.0, -4.0, 6.0])
    assert torch.equal(plain.held(x), want)
    big = torch.zeros(32)
    big[0], big[1] = 7.9, 0.2           # the scale is 1: beyond 6 is 6, and 0.2 is nothing
    assert plain.held(big)[0] == 6 and plain.held(big)[1] == 0
    big[3] = float("inf")
    assert torch.isnan(plain.held(big)).all()


def test_plain_tables_refuse_from_the_first_request_that_does_not_fit():
    table = [[7, -1], [-1, -1], [-1, -1], [9, 8], [-1, -1]]
    found = plain.step_tables([4, 0, 0, 16, 0], [3, 9, 17, 0, 2], table, 8, [5, 6, 3], 0, 20)
    # request 1 takes two pages, request 2 exceeds its row, request 3 is full and brings nothing
    assert found["progress"] == [3, 1]
    assert found["offsets"] == [0, 3, 12, 12, 12, 14]
    assert found["slots"][:3] == [60, 61, 62] and found["slots"][3] == 40 and found["slots"][11] == 48
    assert found["slots"][12:14] == [24, 25] and found["slots"][14:] == [-1] * 6
    assert table == [[7, -1], [5, 6], [-1, -1], [9, 8], [3, -1]]
    table = [[-1], [-1], [-1]]
    found = plain.step_tables([0, 0, 0], [2, 2, 2], table, 8, [1], 0, 20)
    assert found["progress"] == [1, 2] and found["offsets"] == [0, 2, 2, 2] and table == [[1], [-1], [-1]]


def test_page_shapes():
    assert Fp4Pages.shapes(3, 2, 16, 96) == ((3, 2, 16, 48), (3, 2, 16, 3), (3, 2, 4, 12, 4, 4), (3, 2, 4, 3, 4))
    for bad in ((0, 2, 16, 96), (3, 0, 16, 96), (3, 2, 12, 96), (3, 2, 2, 96), (3, 2, 16, 80), (3, 2, 16, 288), (3, 2, 16, 0)):
        with pytest.raises(KernelError):
            Fp4Pages.shapes(*bad)
    with pytest.raises(kernel_build.BuildError):
        kernel_build.build_fp4_attention(48)


def test_tensors_on_the_host_are_refused():
    k = kernels()
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pages = Fp4Pages.empty(2, 1, 16, 32, device="cpu")
    with pytest.raises(KernelError, match="step_tables"):
        k.step_tables(i(2), i(2), i(2, 2), 16, i(4), i(1), i(8), i(8), i(8), i(3), i(2), i(2))
    with pytest.raises(KernelError, match="pages in 4 bits"):
        k.fp4_write(torch.zeros(2, 32), torch.zeros(2, 32), i(2), pages)
    with pytest.raises(KernelError, match="pages in 4 bits"):
        k.fp4_read(pages, i(2), torch.zeros(2, 32), torch.zeros(2, 32))
    with pytest.raises(KernelError, match="pages in 4 bits"):
        k.fp4_attention(torch.zeros(2, 32), 1, 1, 32, pages, i(1, 2), i(2), i(1), 2, 8, torch.zeros(2, 32), 1.0)
    with pytest.raises(KernelError, match="logits"):
        k.token_logprobs(torch.zeros(2, 9), i(2), torch.zeros(2), torch.zeros(2), i(2), i(2, 0), torch.zeros(2, 0))


def test_the_plan_of_the_splits_covers_every_request():
    """The launch's bounds (how many splits there are room and workgroups for) hold for every shorter request: the rule
    of csrc/fp4_attention.hip in whole numbers."""
    def shortest(span, heads):
        return 256 if heads < 4 else 512 if span <= 4096 else 1024

    def decode_split(span, heads):
        return 768 if span <= 768 else max(shortest(span, heads), (-(-span * heads // 512) + 127) // 128 * 128)

    def prompt_split(span, groups, heads):
        want = max(1, 512 // (max(1, groups) * heads))
        return max(256, ((span + want - 1) // want + 63) // 64 * 64)

    def planned(span, heads):
        return 1 if span <= 768 else min(max(-(-n // shortest(n, heads)) for n in (span, min(span, 4096))), -(-512 // heads))

    spans = list(range(0, 5000, 7)) + list(range(32000, 34000, 13)) + list(range(130000, 1100000, 1709)) + [131072, 131073, 262144, 262145]
    for heads in (1, 2, 3, 4, 5, 8, 12, 64, 300, 600):
        worst = 0
        for span in sorted(spans):
            worst = max(worst, -(-span // decode_split(span, heads)))
            assert worst <= planned(span, heads) <= 512, (span, heads)
            for groups in (1, 2, 3, 5, 11, 16, 31, 32, 33, 500):
                many = -(-span // prompt_split(span, groups, heads))
                assert many <= max(1, min(512 // heads, -(-span // 256)))
                assert groups * many <= max(1, 512 // heads) or many <= 1


@pytest.mark.parametrize("rows,requests,heads,group,most,longest", [
    (160, 40, 8, 4, 160, 8192), (65, 65, 8, 1, 1, 8192), (5000, 65, 8, 4, 256, 8192), (4500, 64, 8, 16, 300, 131072)])
def test_memory_of_large_steps_is_counted_in_64_bits(rows, requests, heads, group, most, longest):
    """A thousand times the rows and requests take a thousand times the memory."""
    lib = ctypes.CDLL(str(kernel_build.build_fp4_attention(128)))
    count = lib.ls_fp4_attention_scratch_bytes
    count.restype = ctypes.c_long
    one = count(1, rows, requests, heads, group, most, longest, 0)
    assert 0 < one < 2 ** 33 and count(1, 1000 * rows, 1000 * requests, heads, group, most, longest, 0) == 1000 * one


def plan_entry(head_dim):
    """(splits, workgroups, launched, entries, room, all entries) of a request in a step, by the library's own host code."""
    lib = ctypes.CDLL(str(kernel_build.build_fp4_attention(head_dim)))
    entry, code = lib.ls_fp4_attention_plan, {torch.float32: 0, torch.bfloat16: 1}
    lib.ls_last_error.restype = ctypes.c_char_p

    def plan(dtype, rows, requests, heads, group, most, longest, window, tokens, length):
        out = (ctypes.c_long * 6)()
        assert entry(code[dtype], rows, requests, heads, group, most, longest, window, tokens, length, out) == 0, lib.ls_last_error()
        return tuple(out)
    return plan


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head_dim", [64, 160, 256])
def test_the_library_launches_enough_for_every_request(head_dim, dtype):
    """What a launch is sized for (workgroups, room for the splits' sums) covers every request that it may hold."""
    plan = plan_entry(head_dim)
    rng = random.Random(head_dim)
    for _ in range(6000):
        heads, group = rng.choice((1, 2, 3, 4, 5, 8, 12, 64, 300, 600)), rng.choice((1, 2, 3, 4, 8, 16, 17, 40))
        requests = rng.choice((1, 2, 7, 64, 300))
        longest = int(2 ** rng.uniform(0, 20.5))
        most = min(longest, int(2 ** rng.uniform(0, 13)))
        rows = most + rng.choice((0, requests - 1, rng.randrange(most * requests)))
        window = rng.choice((0, 0, 1, int(2 ** rng.uniform(0, 20))))
        window = 0 if window >= longest else window
        for tokens in {1, most, max(1, min(most, 16 // group)), min(most, 16 // group + 1), rng.randint(1, most), rng.randint(1, min(most, 40))}:
            for length in {longest, tokens, rng.randint(tokens, longest), min(longest, tokens + 4096)}:
                case = (dtype, rows, requests, heads, group, most, longest, window, tokens, length)
                splits, groups, launched, entries, room, held = plan(*case)
                assert 1 <= splits <= groups <= launched, case
                assert splits == 1 or 0 < entries <= room <= held, case
                assert splits <= 512 and (splits - 1) * 256 < length, case


@pytest.mark.parametrize("heads", [511, 512, 600, 1024])
def test_the_longest_requests_of_many_heads_have_their_splits(heads):
    plan = plan_entry(128)
    for longest in (2 ** 29, 2 ** 30 + 12345, 2 ** 31 - 2 ** 16):
        for tokens in (1, 3, 40):
            splits, groups, launched, entries, room, held = plan(torch.bfloat16, 40, 2, heads, 4, 40, longest, 0, tokens, longest)
            assert 1 <= splits <= groups <= launched and entries <= room <= held, (longest, tokens)


def test_areas_that_share_memory():
    from lockstep_amd.ops.kernels import _area, _meet

    buffer = torch.arange(6 * 40).reshape(6, 40)
    rng = random.Random(2)

    def window(strides):
        first, last = sorted(rng.sample(range(7), 2))
        left, right = sorted(rng.sample(range(41), 2))
        x = buffer[first:last, left:right]
        return (x, x) if strides is None else (x[::strides], x[::strides])

    exact = met = 0
    for _ in range(4000):
        kind = rng.choice((None, None, 2))
        (a, _), (b, _) = window(None), window(kind)
        shared = bool(set(a.reshape(-1).tolist()) & set(b.reshape(-1).tolist()))
        found = _meet(_area(a, a.shape[1]), _area(b, b.shape[1]))
        assert found == _meet(_area(b, b.shape[1]), _area(a, a.shape[1]))
        assert found or not shared
        if kind is None and a.shape[0] > 1 and b.shape[0] > 1:
            exact, met = exact + 1, met + shared
            if a.shape == b.shape and a.storage_offset() // 40 == b.storage_offset() // 40:     # the same rows: never refused in vain
                assert found == shared
    assert exact > 1000 and met > 300
    x = torch.zeros(10)
    assert _meet(_area(x), _area(x[9:])) and not _meet(_area(x[:9]), _area(x[9:])) and not _meet(_area(x), _area(x[:0]))
    assert _meet(_area(x[2:3].expand(4, 3), 3), _area(x)) and not _meet(_area(x[:0].reshape(0, 3), 3), _area(x))


def test_splits_leave_no_more_sums_than_they_read_keys():
    """With bfloat16 operands a request of up to 256 rows a head leaves at most what its keys and values take in their pages, but
    for one split's sums (the last split is shorter than the others)."""
    plan = plan_entry(128)
    for group in (1, 2, 4, 8, 16):
        for tokens in {t for t in (1, 3, 5, 9, 17, 20, 33, 64, 100, 256) if t * group <= 256}:
            for length in (300, 800, 1000, 2100, 4096, 8192, 32768, 131072):
                for heads in (1, 2, 8):
                    splits, _, _, entries, _, _ = plan(torch.bfloat16, 256, 4, heads, group, 256, length, 0, tokens, length)
                    rows = tokens * group
                    assert splits == 1 or (entries - rows) * (128 + 2) * 4 <= length * 128 * 17 // 16, (group, tokens, length, heads)


@pytest.mark.parametrize("rows,requests,most,longest", [(64 * 33, 64, 33, 8192), (63 + 2048, 64, 2048, 8192), (255 + 2048, 256, 2048, 32768),
                                                        (255 + 8192, 256, 8192, 131072), (64, 64, 1, 8192)])
def test_memory_of_a_step_is_less_than_its_pages(rows, requests, most, longest):
    """The splits' sums of many short portions, and of a prompt beside decoded tokens, against the pages of such requests (32 heads
    over 8 of 128): a third more at most, where many requests may be of a few tokens behind 8,192 keys."""
    lib = ctypes.CDLL(str(kernel_build.build_fp4_attention(128)))
    count = lib.ls_fp4_attention_scratch_bytes
    count.restype = ctypes.c_long
    pages = requests * longest * 8 * 128 * 17 // 16
    assert 0 < count(1, rows, requests, 8, 4, most, longest, 0) <= pages * 4 // 3


def test_a_library_is_whole_for_the_thread_that_finds_it(monkeypatch):
    """While one thread loads the library, another one that asks for it gets its limits too."""
    from lockstep_amd.ops.kernels import Kernels

    k = Kernels.__new__(Kernels)
    k._serving = k._calls = None
    failed, asked = [], []

    def other():
        try:
            assert k.serving is not None and len(k._serving_limits) == 3
        except Exception as exc:  # noqa: BLE001 - reported below
            failed.append(exc)

    real = ctypes.CDLL

    class Library:
        """The library, whose first call lets another thread in (as every call does that releases the interpreter's lock)."""

        def __init__(self, path):
            self.__dict__["lib"] = real(path)

        def __getattr__(self, name):
            if name == "ls_step_tables_max_requests" and not asked:
                asked.append(threading.Thread(target=other))
                asked[0].start()
                asked[0].join()
            return getattr(self.lib, name)

    monkeypatch.setattr(ctypes, "CDLL", Library)
    assert k.serving is not None
    assert len(asked) == 1 and not failed, failed


def test_pages_are_fp4_pages():
    k = kernels()
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for pages in (tuple(Fp4Pages.empty(2, 1, 16, 32, device="cpu")), list(Fp4Pages.empty(2, 1, 16, 32, device="cpu")), None):
        for call in (lambda: k.fp4_write(torch.zeros(2, 32), torch.zeros(2, 32), i(2), pages),
                     lambda: k.fp4_read(pages, i(2), torch.zeros(2, 32), torch.zeros(2, 32)),
                     lambda: k.fp4_attention(torch.zeros(2, 32), 1, 1, 32, pages, i(1, 2), i(2), i(1), 2, 8, torch.zeros(2, 32), 1.0)):
            with pytest.raises(KernelError, match="Fp4Pages"):
                call()


def test_checked_calls_without_a_compiler_of_the_system(monkeypatch, tmp_path):
    """With hipcc alone the module is built by the compiler that comes with it."""
    from importlib.machinery import ExtensionFileLoader
    from importlib.util import module_from_spec, spec_from_loader

    hipcc = kernel_build.find_hipcc()
    monkeypatch.delenv("CXX", raising=False)
    monkeypatch.setenv("HIPCC", hipcc)
    monkeypatch.setattr(kernel_build.shutil, "which", lambda name: None)
    monkeypatch.setattr(kernel_build, "lib_dirs", lambda: [tmp_path])
    path = kernel_build.build_calls(force=True)
    loader = ExtensionFileLoader("lockstep_calls", str(path))
    module = module_from_spec(spec_from_loader("lockstep_calls", loader))
    loader.exec_module(module)
    assert module.fp4_write(0, 0, torch.zeros(1), torch.zeros(1), torch.zeros(1), None) is False


def test_a_build_goes_on_without_the_checked_calls(monkeypatch, capsys):
    made = []

    def stub(name):
        def build(*args, **kwargs):
            made.append(name)
            return Path(name)
        return build

    for name in dir(kernel_build):
        if name.startswith("build_") and name not in ("build_all", "build_calls_if_possible"):
            monkeypatch.setattr(kernel_build, name, stub(name))

    def fails(force=False):
        raise kernel_build.BuildError("no Python.h")

    monkeypatch.setattr(kernel_build, "build_calls", fails)
    paths = kernel_build.build_all()
    assert len(paths) == len(made) > 20 and all(isinstance(p, Path) for p in paths)
    assert "no Python.h" in capsys.readouterr().err
    monkeypatch.setattr(kernel_build, "build_serving", fails)
    with pytest.raises(kernel_build.BuildError):
        kernel_build.build_all()
