"""The CLI loop with top-k, top-p and min-p: the device's filtered draws of each step against the 64-bit definition on
the same logits, one token left as greedy, and the flags of `python -m inference_engine_rust_amd`."""
import random

import numpy as np
import pytest

import paged_ref
from inference_engine_rust_amd import engine as E
from inference_engine_rust_amd import frontend as F
from test_gpu_frontend import c0_tok  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def parts(c0_tok):
    path, tj, g, eos_at = c0_tok
    return E.LoadedModel.load(path), F.Tokenizer.load_from_file(tj), " ".join(f"w{i}" for i in g["prompt"]), g, eos_at


@pytest.mark.parametrize("top_k,top_p,min_p", [(5, 1.0, 0.0), (0, 0.7, 0.0), (0, 1.0, 0.2), (200, 0.9, 0.01)])
def test_generate_draws_from_what_the_filters_leave(gpu, c0_tok, top_k, top_p, min_p):
    m, tok, prompt, g, _ = parts(c0_tok)
    _, ids = F.generate(m, tok, prompt, new_tokens=8, temperature=0.9, rng=random.Random(3), top_k=top_k, top_p=top_p, min_p=min_p)
    s = E.InferenceSession(m)
    s.prefill(np.array(g["prompt"], np.uint32))
    eos, draws, want = m.tokenizer_prompt().eos_token_id, random.Random(3), []
    for _ in range(8):
        pick, _ = paged_ref.sample(s.logits_last_token(), 0.9, draws.random(), top_k, top_p, min_p)
        if pick == eos:
            break
        want.append(pick)
        s.decode_token(pick)
    assert ids == want


def test_one_token_left_is_greedy(gpu, c0_tok):
    m, tok, prompt, g, eos_at = parts(c0_tok)
    for kw in ({"top_k": 1}, {"top_p": 0.0}, {"min_p": 1.0}):
        _, ids = F.generate(m, tok, prompt, new_tokens=6, temperature=1.3, rng=random.Random(0), **kw)
        assert ids == g["tokens"][:min(6, eos_at)], kw


def test_cli_flags(gpu, c0_tok, capsys):
    path, tj, g, eos_at = c0_tok
    prompt = " ".join(f"w{i}" for i in g["prompt"])
    run = ["-m", path, "-t", tj, "-n", "6", "--temperature", "0.7"]
    assert F.main(run + ["--top-k", "1", prompt]) == 0
    assert capsys.readouterr().out.strip() == " ".join(f"w{i}" for i in g["tokens"][:min(6, eos_at)])
    assert F.main(run + ["--top-p", "nan", prompt]) == 1
    assert "NaN" in capsys.readouterr().err
