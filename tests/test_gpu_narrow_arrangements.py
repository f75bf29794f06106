"""Every small model with 4-bit weights, through the engine, against itself with the matrices that these weights stand for."""
import importlib

import numpy as np
import pytest
import torch

import narrow_util as U
import qstream_b200 as qs
from qstream_b200.csrc.q4 import Weight4
from qstream_b200.parts import Part
from test_narrow_arrangements import MODELS, WIDE_ONLY
from util import random_tokens
from vofinex_util import assert_close

pytestmark = pytest.mark.gpu


def widen(part):
    """Replace every 4-bit matrix that `part` and what it is made of hold by a float32 one, exactly; how many."""
    n = 0
    for name, value in list(vars(part).items()):
        if isinstance(value, Weight4):
            setattr(part, name, torch.from_numpy(U.dense(value).astype(np.float32)).cuda())
            n += 1
        elif isinstance(value, Part):
            n += widen(value)
    return n


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,which", [m for m in MODELS if m not in WIDE_ONLY])
def test_narrow_matrices_are_the_matrices_they_stand_for(tmp_path, name, which, dtype):
    """Two sequences: prompts, one of them in two portions, then single tokens.  The products differ in the order of 32-bit sums: as the families' engines differ
    from their plain models."""
    folder, _ = importlib.import_module(name + "_util").make_folder(tmp_path, which, dtype)
    narrow, wide = (qs.load_model(folder, dtype=dtype, weight_bits=4, weight_group=32) for _ in range(2))
    assert sum(widen(block) for block in wide.blocks) == len(narrow.runtime.narrowed) > 0
    rng = np.random.default_rng(7)
    prompts = [random_tokens(rng, 70, narrow.vocab_size), random_tokens(rng, 21, narrow.vocab_size)]
    later = [random_tokens(rng, 2, narrow.vocab_size) for _ in range(6)]

    def logits(model):
        engine = qs.Engine(model, max_tokens=512, max_batch=2)
        slots = [engine.acquire(), engine.acquire()]
        got = [engine.step(slots, [prompts[0][:40], prompts[1]], [list(range(40)), list(range(21))]).cpu().numpy(),
               engine.step([slots[0]], [prompts[0][40:]], [list(range(30))]).cpu().numpy()]
        got += [engine.step(slots, [[t] for t in toks]).cpu().numpy() for toks in later]
        engine.check_status()
        return np.concatenate(got)

    assert_close(logits(narrow), logits(wide), dtype, f"{name} {which}")
