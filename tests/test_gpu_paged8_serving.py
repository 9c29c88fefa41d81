# SPDX-License-Identifier: Apache-2.0
"""The serving example with rotary positions and the cache in 8 bits runs, with
more requests than slots, pages reused and a captured generation step."""
import pytest
import torch

from examples.paged_serving import serve

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [None, "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_example_runs(kv, dtype):
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(500, (n,), generator=g).tolist() for n in (40, 7, 1, 100, 16, 33)]
    generated, last, model = serve(prompts, 9, dtype=dtype, rotary=True, kv=kv, slots=3, num_pages=24)
    assert [len(x) for x in generated] == [9] * len(prompts)
    for x in last:
        assert x.shape == (500,) and torch.isfinite(x).all()
