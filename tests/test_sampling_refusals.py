"""Shapes that the sampling kernels cannot take are refused where their workspace is sized, which every caller of theirs asks
for first: the device entry, the host entry and a session (of a vocabulary as large)."""
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
