"""Rotations of more heads than a launch has rows of CTAs: four targets of up
to 65535 heads each, against the rotation of each target alone."""
import pytest

import neon_cuda as N

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dim,rot,half,heads", [
    (1024, 64, False, [65535] * 4),   # pieces of two values: two heads a CTA
    (1024, 64, True, [65535] * 3),    # one
    (600, 16, False, [65535] * 4),    # three
    (16, 16, True, [65535] * 4)])
def test_more_heads_than_grid_rows(dim, rot, half, heads):
    N.init(0)
    spec = N.Rope(rot, half=half)
    pos = torch.tensor([77], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    # not on 16 bytes: single values or pairs
    x = [torch.randn(h * dim + 1, generator=g, device="cuda").bfloat16()[1:] for h in heads]
    y = [torch.empty(h * dim + 1, dtype=torch.bfloat16, device="cuda")[1:].fill_(9) for h in heads]
    N.rope(spec, pos, 1, dim, list(zip(x, y, heads)), type=N.GGML_BF16)
    for a, b, h in zip(x, y, heads):
        alone = torch.empty_like(a)
        N.rope(spec, pos, 1, dim, [(a, alone, h)], type=N.GGML_BF16)
        assert torch.equal(b, alone)
    few = torch.empty(5 * dim, dtype=torch.bfloat16, device="cuda")
    N.rope(spec, pos, 1, dim, [(x[-1][-5 * dim:], few, 5)], type=N.GGML_BF16)
    assert torch.equal(few, y[-1][-5 * dim:])
