"""The rotation with every value that a table can hold."""
import numpy as np
import pytest
import torch

from oracle import paged as o_paged
from test_gpu_paged import _bf16, _gpu, _kernel, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,rotary", [(32, 32), (64, 32), (128, 128)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("scaled", [False, True])
def test_append_with_tables_of_any_int16(stream, D, rotary, adjacent, scaled):
    """-2^15 has no negative of 16 bits; codes of -128 beside it."""
    H, Hk, page, T = 4, 2, 16, 40
    rng = np.random.default_rng([3, D])
    table, n_pages = _table(rng, page, [T])
    rope = rng.choice(np.array([-32768, -32767, -16385, -1, 0, 1, 11585, 16384, 32767], dtype=np.int16), (T, rotary // 2, 2))
    if scaled:
        q, kv = _bf16(rng, T, H * D), _bf16(rng, T, 2 * Hk * D)
    else:
        q, kv = (torch.from_numpy(rng.choice(np.array([-128, -127, -64, -1, 0, 1, 90, 127], dtype=np.int8), (T, w))) for w in (H * D, 2 * Hk * D))
    kern = _kernel(H, Hk, D, page, rotary=rotary, adjacent=adjacent)
    pages, scales, q_out = kern.pages(n_pages), kern.page_scales(n_pages), torch.zeros((T, H * D), dtype=torch.int8, device="cuda")
    q_scale, pos = torch.zeros((T, H), device="cuda"), np.arange(T, dtype=np.int32)
    args = [_gpu(a) for a in (q, kv, np.zeros(T, dtype=np.int32), pos, table)]
    t_rope = _gpu(rope)
    torch.cuda.synchronize()
    if scaled:
        kern.append_scaled(stream, *args, pages, scales, q_out, q_scale, t_rope)
    else:
        kern.append(stream, *args, pages, q_out, t_rope)
    stream.synchronize()
    stored = pages.cpu().numpy()[table[0, pos // page], :, pos % page, :D]
    stored_scale = scales.cpu().numpy()[table[0, pos // page], :, pos % page, 0]
    for x, got, got_scale in ((q.view(T, H, D), q_out.cpu().numpy().reshape(T, H, D), q_scale.cpu().numpy()),
                              (kv.view(T, Hk, 2, D)[:, :, 0], stored, stored_scale)):
        want = o_paged.rotate(np.ascontiguousarray(x.float().numpy() if scaled else x.numpy()), rope, rotary, adjacent)
        if scaled:
            want, want_scale = o_paged.quantise(want)
            assert np.array_equal(got_scale, want_scale)
        assert np.array_equal(got, want)
