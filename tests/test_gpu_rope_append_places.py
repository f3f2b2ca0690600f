"""Tables of no positions, in the append: no token has a place."""

import pytest
import torch

from testt_amd import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch", [0, 1, 3])
def test_tables_of_no_positions(batch, interleaved):
    d = 32
    pages = torch.full((2, 4, 1, 4, d), 7.0, dtype=torch.float16, device=DEV)
    qkv = torch.randn(3, 4 * d, generator=torch.Generator().manual_seed(1)).to(torch.float16).to(DEV)
    cos, sin = rope.rotary_tables(0, d, device=DEV)
    table = torch.arange(batch, dtype=I32, device=DEV).view(batch, 1)
    cu = torch.tensor([0, 1, 2, 3][:batch + 1], dtype=I32, device=DEV)
    q = rope.rope_append(qkv, None, None, cos, sin, pages[0], pages[1], table, torch.ones(batch, dtype=I32, device=DEV),
                         cu, interleaved)
    assert not bool(q.any()) and bool((pages == 7).all())
    # as with tables that end before the token's position
    full = rope.rotary_tables(4, d, device=DEV)
    q = rope.rope_append(qkv, None, None, full[0][:0], full[1][:0], pages[0], pages[1], table,
                         torch.ones(batch, dtype=I32, device=DEV), cu, interleaved)
    assert not bool(q.any()) and bool((pages == 7).all())
