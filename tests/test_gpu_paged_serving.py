# SPDX-License-Identifier: Apache-2.0
"""The serving example end to end: prompts, a captured generation step, page
reuse, against a recomputation without any cache (GPU)."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "paged_serving.py"


@pytest.mark.parametrize("dtype,hq,hkv,d,page,pages", [
    (torch.bfloat16, 8, 2, 64, 16, 26),     # pages for two or three requests at a time
    (torch.float16, 4, 4, 72, 8, 200),
])
def test_serving_matches_recomputation(dtype, hq, hkv, d, page, pages):
    spec = importlib.util.spec_from_file_location("paged_serving", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(300, (n,), generator=g).tolist() for n in (5, 130, 16, 1, 64, 200, 33)]
    generated, last, model = example.serve(prompts, 9, vocab=300, hq=hq, hkv=hkv, d=d, page_size=page, num_pages=pages,
                                           slots=3, dtype=dtype)
    for prompt, answer, got in zip(prompts, generated, last):
        assert len(answer) == 9 and answer[-1] == int(got.argmax())
        with torch.inference_mode():
            want = model.forward(torch.tensor(prompt + answer[:-1], device="cuda"))
        # about 12 roundings of unit-size 16-bit activations on each side, the
        # largest of 300 logits: 4 sqrt(24) = 20 unit roundoffs, and a margin
        unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
        assert (got - want).abs().max().item() <= 32 * unit, (len(prompt), (got - want).abs().max().item())
