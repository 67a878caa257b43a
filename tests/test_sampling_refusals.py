"""Shapes that the sampling kernels cannot take are refused where their workspace is sized, which every caller of theirs asks
for first: the device entry, the host entry and a session (of a vocabulary as large)."""
import ctypes
import pathlib
import re

import pytest

from inference_engine_rust_amd import engine as E

CSRC = pathlib.Path(__file__).resolve().parent.parent / "inference_engine_rust_amd" / "csrc"


def test_workspace_sizes_refuse():
    for rows, n, kind in ((1, 0, "Sampling"), (0, 0, "Sampling"), (1, 2 ** 25 + 1, "Op"), (2 ** 21 + 1, 5, "Op"), (0, 2 ** 25 + 1, "Op")):
        with pytest.raises(E.EngineError) as e:
            E.sample_workspace(rows, n)
        assert e.value.kind == kind
    assert E.sample_workspace(2 ** 21, 2 ** 15) == 0 < E.sample_workspace(1, 2 ** 15 + 1) < E.sample_workspace(1, 2 ** 25)


@pytest.mark.parametrize("path", ["api.cpp", "session.cpp"])
def test_every_launch_is_behind_a_workspace_size(path):
    """(A model with a vocabulary beyond 2^25 would be needed to reach the session's: read from the source.)"""
    text = (CSRC / path).read_text()
    for at in (m.start() for m in re.finditer(r"\blaunch_sample\(", text)):
        body = text[max(text.rfind("\n}\n", 0, at), 0):at]  # (the function so far)
        size = re.search(r"(const size_t [^;]*|\b)= sample_workspace\([^;]*\);", body)
        assert size and "if (" not in body[body.rfind("\n", 0, size.start()) + 1:size.start()], body


class Entries:
    """In the library's place: what its entries are given, through their declared types."""

    def __init__(self):
        self.given = []

    def __getattr__(self, name):
        def entry(*args):
            self.given.append([t(a).value if t in (ctypes.c_float, ctypes.c_int32) else None for t, a in zip(E.EXPORTS[name][0], args)])
            return 0
        return entry


@pytest.mark.parametrize("top_k,held", [(0, 0), (-1, 0), (50, 50), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1), (-2 ** 32 - 5, 0)])
@pytest.mark.parametrize("r", [0.0, 0.3, 1 - 2.0 ** -24, 1 - 2.0 ** -25, 1 - 2.0 ** -53])
def test_draws_below_one_and_any_top_k_arrive_as_such(monkeypatch, r, top_k, held):
    """A draw of 64 bits next to 1 is no 1 in 32, and a top_k of more bits than 32 keeps its meaning."""
    entries = Entries()
    monkeypatch.setattr(E, "lib", lambda: entries)
    E.host_sample([1.0], 1.0, r, top_k)
    E.sample_next_token(type("Session", (), {"_h": None}), 1.0, r, top_k)
    (_, _, _, k0, _, _, r0, _, _), (_, _, k1, _, _, r1, _) = entries.given
    assert k0 == k1 == held and r0 == r1 < 1 and abs(r0 - r) <= 2.0 ** -24


@pytest.mark.parametrize("r", [1.0, 2.0, -0.1])
def test_other_draws_go_on_to_be_refused(monkeypatch, r):
    entries = Entries()
    monkeypatch.setattr(E, "lib", lambda: entries)
    E.host_sample([1.0], 1.0, r)
    assert not 0 <= entries.given[0][6] < 1
