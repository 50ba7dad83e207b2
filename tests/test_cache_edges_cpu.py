"""Refusals of the operators around a key-value cache that protect memory and results, and the build of their module,
without a device: the C entries check every argument before their first CUDA call."""
import ctypes

import pytest
import torch

from intent_b200 import _native
from test_cache_operators_cpu import FAR, SPACE, attend, backward, rotary, view, write

needs_no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="would launch")
ACCEPTED = _native.ERR_CUDA      # all checks passed: the launch fails where there is no device


# ------------------------------------------------------------------------------- overlaps
@pytest.mark.parametrize("change", [
    {"qw": view(64, address=FAR[2] + 512)}, {"kw": view(64, address=FAR[3])}, {"cos": view(100, 32, address=FAR[2] - 64)},
    {"sin": view(100, 32, address=FAR[3] - 12800 + 16)}, {"positions": view(5, address=FAR[2] + 4)},
    {"space": view(64, address=FAR[2])}, {"space": view(64, address=FAR[0] + 128)}])
def test_rotary_outputs_overlap_no_operand(change):
    assert rotary(**change) == 1


@pytest.mark.parametrize("change", [
    {"dkw": view(64, address=FAR[6])}, {"dkw": view(64, address=FAR[6] + 252)}, {"dqw": view(64, address=FAR[2] + 4)},
    {"dqw": view(64, address=FAR[0])}, {"qw": view(64, address=FAR[7])}, {"positions": view(5, address=FAR[8] + 32)},
    {"cos": view(100, 32, address=FAR[2])}, {"space": view(64, address=FAR[8])}, {"dkw": view(64, address=FAR[8] + 16)}])
def test_rotary_gradients_overlap_no_operand(change):
    assert backward(**change) == 1


@pytest.mark.parametrize("change", [
    {"ks": view(3, 2, 16, address=FAR[2] + 512)}, {"vs": view(3, 2, 16, address=FAR[2])}, {"ks": view(3, 2, 16, address=FAR[3] + 6140)},
    {"slots": view(6, address=FAR[2])}, {"slots": view(6, address=FAR[5] + 8)}, {"space": view(64, address=FAR[2] + 64)},
    {"space": view(64, address=FAR[4])}, {"space": view(64, address=FAR[0])},
    # inside each page, but over the codes' last row
    {"kc": view(3, 2, 16, 64, address=FAR[2], strides=[4096, 1024, 64, 1]), "ks": view(3, 2, 16, address=FAR[2] + 2044, strides=[1024, 16, 1])}])
def test_what_cache_write_writes_overlaps_no_operand(change):
    assert write(**change) == 1


@needs_no_device
def test_scales_beside_their_codes_are_taken_apart():
    """One allocation for codes and scales: page for page, and row for row."""
    for heads, page in ((2, 16), (1, 1), (3, 5)):
        body = heads * page * 64
        pitch = 2 * body + 2 * heads * page * 4
        pitch += -pitch % 16
        at = [FAR[2], FAR[2] + body, FAR[2] + 2 * body, FAR[2] + 2 * body + heads * page * 4]
        codes = [view(3, heads, page, 64, address=x, strides=[pitch, page * 64, 64, 1]) for x in at[:2]]
        scales = [view(3, heads, page, address=x, strides=[pitch // 4, page, 1]) for x in at[2:]]
        rows = view(6, heads, 64, address=FAR[0]), view(6, heads, 64, address=FAR[1])
        assert write(k=rows[0], v=rows[1], kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1]) == ACCEPTED
        row = 2 * (64 + 16)
        codes = [view(3, heads, page, 64, address=FAR[2] + x, strides=[page * heads * row, row, heads * row, 1]) for x in (0, 64)]
        scales = [view(3, heads, page, address=FAR[2] + x, strides=[page * heads * row // 4, row // 4, heads * row // 4]) for x in (128, 132)]
        assert write(k=rows[0], v=rows[1], kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1]) == ACCEPTED
        scales[1][0] -= 4                                    # on the other's
        assert write(k=rows[0], v=rows[1], kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1]) == 1
        scales[1][0] = FAR[2] + 124                          # over the last codes of v
        assert write(k=rows[0], v=rows[1], kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1]) == 1


def test_what_cache_read_writes_overlaps_no_operand():
    read = "b200_cache_read"
    assert write(read, slots=view(6, address=FAR[0] + 8)) == 1 and write(read, slots=view(6, address=FAR[1])) == 1
    assert write(read, space=view(64, address=FAR[1] + 256)) == 1 and write(read, space=view(64, address=FAR[3])) == 1
    assert write(read, space=view(64, address=FAR[5])) == 1


@pytest.mark.parametrize("change", [
    {"lse": view(2, 8, address=FAR[3])}, {"lse": view(2, 8, address=FAR[0] + 4)}, {"lse": view(2, 8, address=FAR[4])},
    {"lse": view(2, 8, address=FAR[5], strides=[0, 1])}, {"lse": view(2, 8, address=FAR[5], strides=[4, 1])},
    {"lse": view(2, 8, address=FAR[1] + 32)}, {"table": view(2, 300, address=FAR[3] + 16)}, {"lengths": view(2, address=FAR[3])},
    {"lengths": view(2, address=FAR[4] + 4)}, {"table": view(2, 300, address=FAR[4])}, {"space": view(64, address=FAR[3])},
    {"space": view(64, address=FAR[2])}, {"q": view(2, 8, 64, address=FAR[4] + 1024)}])
def test_what_paged_attention_writes_overlaps_no_operand(change):
    assert attend(**change) == 1


def test_scales_that_attention_writes_over_are_refused():
    codes = {"store": 3, "ks": view(9, 2, 16, address=FAR[6]), "vs": view(9, 2, 16, address=FAR[7])}
    for place in (FAR[6] + 128, FAR[7]):
        assert attend(**codes, out=view(2, 8, 64, address=place)) == 1
        assert attend(**codes, lse=view(2, 8, address=place)) == 1
    if not torch.cuda.is_available():
        assert attend(**codes) == ACCEPTED and attend(lse=view(2, 8, address=FAR[5])) == ACCEPTED


# ------------------------------------------------------------------------------ alignment
@pytest.mark.parametrize("call, change", [
    (rotary, {"positions": view(5, address=FAR[9] + 2)}), (rotary, {"space": view(64, address=FAR[9] + 1)}),
    (backward, {"positions": view(5, address=FAR[9] + 1)}), (backward, {"dqw": view(64, address=FAR[9] + 2)}),
    (backward, {"dkw": view(64, address=FAR[9] + 1)}), (backward, {"partial": view(64, 64, address=FAR[9] + 2)}),
    (write, {"space": view(64, address=FAR[9] + 2)}), (attend, {"table": view(2, 300, address=FAR[9] + 2)}),
    (attend, {"lengths": view(2, address=FAR[9] + 1)}), (attend, {"lse": view(2, 8, address=FAR[9] + 2)}),
    (attend, {"space": view(64, address=FAR[9] + 3)})])
def test_words_that_are_not_aligned_are_refused(call, change):
    """A kernel that loads one of them would fault."""
    assert call(**change) == 2


def test_views_whose_reach_passes_64_bits_are_refused():
    """Each axis is in range, but all of them together reach 2^63 bytes, where the comparison of places would wrap."""
    huge = 1 << 30
    cache = view(huge, 1, huge, 64, address=FAR[2], strides=[0, 0, 64, 1])
    scales = view(huge, 1, huge, address=FAR[4], strides=[huge, 0, huge])
    rows = [view(6, 1, 64, address=x) for x in FAR[:2]]
    assert write("b200_cache_read", k=rows[0], v=rows[1], kc=cache, vc=cache, ks=scales, vs=scales) == 1


# ------------------------------------------------------------------------- the native module
def test_the_module_is_rebuilt_for_another_torch(monkeypatch, tmp_path):
    """Its source is older than it, but it was built against other headers."""
    from intent_b200 import build
    module, commands = tmp_path / "binding.so", []

    def compile(command):
        commands.append(command)
        module.write_bytes(f"... built for {_native.binding_built_for()};".encode())
        return ""
    monkeypatch.setattr(build, "BINDING", module)
    monkeypatch.setattr(build, "_run", compile)
    for expected in (1, 1):
        build.build_binding()
        assert len(commands) == expected
    real = _native.binding_built_for()
    monkeypatch.setattr(_native, "binding_built_for", lambda: real.replace("torch ", "torch 9"))
    for expected in (2, 2):
        build.build_binding()
        assert len(commands) == expected


def test_a_module_built_for_another_torch_is_not_loaded(monkeypatch, tmp_path):
    from intent_b200 import tools
    module = tmp_path / "binding.so"
    monkeypatch.setattr(_native, "BINDING_PATH", module)
    monkeypatch.setattr(_native, "_binding", None)
    for content in ("", "built for torch 1.0 0 python cpython-27;"):
        module.write_text(content)
        with pytest.raises(_native.NativeLibraryMissing, match="build it again"):
            _native.binding()
    # the library is there all the same, and doctor says which of the two is not
    report = {entry["name"]: entry for entry in tools.doctor(None)["checks"]}
    assert report["native library"]["status"] == "available" and report["native binding"]["status"] == "unavailable"
    monkeypatch.undo()
    report = {entry["name"]: entry for entry in tools.doctor(None)["checks"]}
    assert "native binding" not in report and report["native library"]["detail"]["binding"] == str(_native.BINDING_PATH)
