"""The example that runs the paged cache's operators together: token by token and as one chunk
its decoder has to give the same states."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from conftest import ROOT  # noqa: E402

spec = importlib.util.spec_from_file_location(
    "cached_decode", os.path.join(ROOT, "examples", "cached_decode.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


@pytest.mark.parametrize("cache", ["int8", "fp16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 4)])
def test_token_by_token_equals_one_chunk(cache, window, sinks):
    """The projections are exact in any batch (int8 products of the same codes); attention's
    fp32 results differ by a few ulp between its two kernels, which the next layer's Q8_0
    quantizer can turn into one code (1/127 of a block's largest value) in rare places."""
    steps, lens = 6, (37, 5, 120)
    a, b = example.run(cache, steps, lens, window, sinks, one_chunk=True)
    for n, s, c in zip(lens, a, b):
        assert s.shape == c.shape == (n + steps, 512) and bool(torch.isfinite(c).all())
        off = (s - c).norm(dim=-1) / c.norm(dim=-1)
        assert float(off.max()) <= 1.0 / 127


def test_requests_do_not_touch_each_other():
    """A request's states do not depend on the requests beside it."""
    a = example.run("fp16", 3, (37, 5, 120))
    b = example.run("fp16", 3, (37,))
    off = (a[0] - b[0]).norm(dim=-1) / b[0].norm(dim=-1)
    assert float(off.max()) <= 1.0 / 127
