# SPDX-License-Identifier: Apache-2.0
"""The serving example with rotary positions, over the cache in 16 bits and in
8, against a recomputation without any cache; and recomputations with planted
mistakes, which have to differ (GPU)."""
import pytest
import torch

from examples.paged_serving import serve
from kotflash_b200 import attention

pytestmark = pytest.mark.gpu

# Of unit-size logits, beyond the 32 unit roundoffs of a recomputation in 16
# bits.  A code's rounding moves an element by a relative r (root mean square): e4m3
# keeps 4 bits, r <= 2^-5; an int8 scale is at most 2 / 127.5 of a row's largest,
# which is within 4 sigma, so a step of 0.063 sigma, r <= 0.018.  Scores and
# values each move an attention's output by r, both layers the logits: 2 sqrt(2)
# r, and the largest of some 3000 logits 4.5 times that.
BEYOND = {None: 0.0, "e4m3": 0.4, "int8": 0.23}


def _recompute(model, tokens, prompt, mistake=None):
    positions = torch.arange(len(tokens), device="cuda")
    if mistake in ("late", "a page late"):  # generated tokens too far
        positions = positions + (positions >= prompt) * (16 if mistake == "a page late" else 1)
    x = model.embed[torch.tensor(tokens, device="cuda")][None]
    rotated = model.heads

    def heads(x, layer, positions):
        q, k, v = rotated(x, layer, positions)
        if mistake == "unrotated":  # the prompt's keys as they were
            frequencies, model.frequencies = model.frequencies, None
            k = torch.cat((rotated(x, layer, positions)[1][:, :, :prompt], k[:, :, prompt:]), 2)
            model.frequencies = frequencies
        return q, k, v

    for layer in range(len(model.qkv)):
        q, k, v = heads(x, layer, positions)
        x = model.residual(x, attention(q, k, v, causal=True), layer)
    return model.logits(x[0, -1])


@pytest.mark.parametrize("kv", [None, "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_matches_recomputation(kv, dtype):
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(500, (n,), generator=g).tolist() for n in (40, 7, 1, 100, 16, 33)]
    generated, last, model = serve(prompts, 9, dtype=dtype, rotary=True, kv=kv, slots=3, num_pages=24)
    bound = BEYOND[kv] + 32 * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11)
    off = {None: [], "late": [], "a page late": [], "unrotated": []}
    for prompt, answer, got in zip(prompts, generated, last):
        assert len(answer) == 9 and answer[-1] == int(got.argmax())
        with torch.inference_mode():
            for mistake, found in off.items():
                found.append((got - _recompute(model, prompt + answer[:-1], len(prompt), mistake)).abs().max().item())
            want = model.forward(torch.tensor(prompt + answer[:-1], device="cuda"))
            assert torch.equal(_recompute(model, prompt + answer[:-1], len(prompt)), want)
    assert max(off[None]) <= bound, off
    # (a prompt of one token knows no difference in its keys' rotation, and one position hides behind 8 bits)
    assert all(max(off[x]) > 2 * bound for x in ("a page late", "unrotated") + (("late",) if kv is None else ())), off
