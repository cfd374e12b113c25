"""attention_join through its C entry point into the memory of one of the parts: out, lse, or both."""
import ctypes

import pytest
import torch

from test_expanded_refusals import _lib, vp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("parts", [1, 2, 4, 7, 32])
@pytest.mark.parametrize("dim", [8, 24, 128, 192, 512, 2048])
def test_a_part_as_the_result(parts, dim):
    """Rows of one warp, of several (dim 512 and more), and such as begin in one warp and end in the next (24, 192): the same as into memory of its own."""
    lib, names = _lib()
    rows = 5000
    gen = torch.Generator(device="cuda").manual_seed(dim + parts)
    outs = [torch.randn(rows, dim, generator=gen, device="cuda").bfloat16() for _ in range(parts)]
    lses = [torch.randn(rows, generator=gen, device="cuda") * 4 for _ in range(parts)]
    for i, lse in enumerate(lses):
        lse[i::5] = float("-inf")

    def join(o, l, out, lse):
        pointers = lambda ts: (vp * parts)(*[t.data_ptr() for t in ts])  # noqa: E731
        assert lib.dsv3_attention_join(pointers(o), pointers(l), parts, rows, dim, out.data_ptr(), lse.data_ptr(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == names.OK

    want, want_lse = torch.empty_like(outs[0]), torch.empty_like(lses[0])
    join(outs, lses, want, want_lse)
    for into in sorted({0, parts // 2, parts - 1}):
        for own_out, own_lse in ((True, False), (False, True), (False, False)):
            o, l = [t.clone() for t in outs], [t.clone() for t in lses]
            out, lse = torch.empty_like(want) if own_out else o[into], torch.empty_like(want_lse) if own_lse else l[into]
            join(o, l, out, lse)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
