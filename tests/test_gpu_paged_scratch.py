"""One scratch buffer for calls of several shapes."""
import numpy as np
import pytest
import torch

from test_gpu_paged import _codes, _gpu, _kernel, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hk,D,most", [(32, 4, 128, 5), (32, 32, 128, 9), (24, 1, 64, 2), (4, 4, 32, 32)])
def test_scratch_for_the_most_tokens_suffices_for_fewer(stream, H, Hk, D, most):
    """A buffer for the most sequences and drafted tokens that a host has: calls of fewer take it, with the results of calls that
    take their own memory."""
    page, B = 64, 3
    rng = np.random.default_rng([9, H, D])
    lens = [4000, 17, 900]
    table, n_pages = _table(rng, page, [n + most for n in lens], room=300000)
    kern = _kernel(H, Hk, D, page)
    pages, t_table, t_lens = _gpu(_codes(rng, n_pages, Hk, page, 2 * D)), _gpu(table), _gpu(np.array(lens, dtype=np.int32))
    sk, sv, temp = _gpu(_codes(rng, H, D)), _gpu(_codes(rng, H, D)), _gpu(np.ones(H, dtype=np.float32))
    scratch = kern.scratch(stream, B, most)
    sizes = [kern.scratch(stream, b, n).numel() for b in (1, B) for n in range(1, most + 1)]
    assert max(sizes) == scratch.numel() and sizes == sorted(sizes[:most]) + sorted(sizes[most:])
    for b in (1, B):
        for n in range(1, most + 1):
            q = _gpu(_codes(rng, b * n, H * D))
            out, own = (torch.zeros((b * n, H * D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            torch.cuda.synchronize()
            kern.decode(stream, q, pages, t_table[:b], t_lens[:b], sk, sv, temp, out, scratch=scratch)
            kern.decode(stream, q, pages, t_table[:b], t_lens[:b], sk, sv, temp, own)
            stream.synchronize()
            assert out.any() and torch.equal(out, own)
