"""The plain default stack against the oracle: a compressed prompt and steps."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from conftest import REL_TOL, max_rel_err
from plain_default_stack import Sequence, tensors
from rustcrates_amd import configs, seeded


@pytest.mark.parametrize("S", [1, 21, 40])
def test_plain_default_stack_is_the_oracles(S):
    V, ctx = 120, 64
    o = configs.build_reference_default(oracle.Network(), V, 5, ctx, wavelet_embedding=False)
    prompt = seeded.prompts(3, [S], V)
    ids, want = o.generate(prompt, n_new=6, want_logits=True)
    s = Sequence(tensors(o, V, ctx))
    got = [s.prompt(prompt[0])] + [s.step(int(t)) for t in ids[0, :-1]]
    assert max_rel_err(np.array(got), np.asarray(want).reshape(6, V)) < REL_TOL
    o.close()
