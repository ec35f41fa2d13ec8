"""The serving operators together (examples/paged_batch.py): batches over the
paged cache decode as the CPU reference does (oracle/llama_ref.py, TR's GPT
step), with ragged prompts and behind a shared first text, and the penalties
act on what is picked."""
import importlib.util
import os
import sys

import numpy as np
import pytest
import torch

import tcb_b200 as T
from tcb_b200 import llama

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from decoder_check import TOL, check_history, fp16_prompt_deviation  # noqa: E402

pytestmark = pytest.mark.gpu

CFG = llama.LlamaConfig(n_layers=2, d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn_dim=1024, vocab=2048, max_ctx=160,
                        eps=1e-5, rope_theta=500000.0)
FIRST = [17, 901, 5, 1333, 42, 2047, 0, 777] * 5
PROMPTS = [FIRST + [3, 99], FIRST + [7], FIRST[:33] + [500, 501], FIRST + [1, 2, 3, 4, 5, 6, 7, 8, 9]]


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_batch.py")
    spec = importlib.util.spec_from_file_location("paged_batch", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def setup(oracle):
    host = llama.host_model(CFG, seed=15, varied=True)
    ctx = T.Context(0)
    # q, the softmax weights and the attention's result are rounded to fp16, and
    # so is one more operand of every product where many rows go through the
    # tensor cores: what that rounding does to the reference, with room for
    # its other draws
    tol = max(TOL, 2.5 * fp16_prompt_deviation(host, np.array(PROMPTS[0])))
    return ctx, host, llama.device_model(CFG, 15, host), tol


@pytest.mark.parametrize("shared,page", [(0, 16), (0, 64), (len(FIRST), 16)])
def test_batch_decodes_as_the_reference(example, setup, shared, page):
    ctx, host, dev, tol = setup
    ctx.device_error(clear=True)
    prompts = PROMPTS if not shared else [PROMPTS[0], PROMPTS[1], PROMPTS[3]]
    batch = example.PagedBatch(ctx, dev, len(prompts), 60, page)
    history, total, logits = example.generate(batch, prompts, 20, shared=shared)
    assert ctx.device_error() == 0
    assert (batch.prefix is not None) == bool(shared)
    for b, p in enumerate(prompts):
        toks = history[b, :int(total[b])].tolist()
        assert toks[:len(p)] == p
        got = {len(p) - 1 + i: lg.cpu().numpy() for i, lg in enumerate(logits[b])}
        check_history(host, toks, len(p), got, tol=tol)


def test_repetition_penalty_changes_what_is_picked(example, setup):
    ctx, _, dev, _ = setup
    rep = torch.full((2,), 50.0, device="cuda")
    history, total, _ = example.generate(example.PagedBatch(ctx, dev, 2, 40), PROMPTS[:2], 20, repetition=rep)
    for b, p in enumerate(PROMPTS[:2]):
        made = history[b, len(p):int(total[b])].tolist()
        assert len(set(made)) == len(made) and not set(made) & set(p)


def test_too_few_pages_are_refused(example, setup):
    ctx, _, dev, _ = setup
    with pytest.raises(RuntimeError):
        example.generate(example.PagedBatch(ctx, dev, 2, 4), PROMPTS[:2], 4)
