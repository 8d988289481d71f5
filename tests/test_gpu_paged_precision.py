"""What the paged decode's bf16 outputs are held to beside the output's own rounding: sums and weights at 32-bit level. The bf16
value has to lie between those of (exact - bound) and (exact + bound), bound counting the roundings in front of the last one."""
import numpy as np
import pytest
import torch

from oracle import paged as o_paged
from test_gpu_paged import _cache, _codes, _gpu, _kernel, _table

pytestmark = pytest.mark.gpu


def _bf16(x):
    return torch.from_numpy(x).to(torch.bfloat16).double().numpy()   # (to nearest, from 64 bits)


def _bound(n, top, mean, v, v_scale, weight_steps):
    """In steps of 2^-24 of the mean |value|: a score's eight roundings, the exponential's 16, the weight's, 64 of joins and the
    division, and for each of two matrix products over 16 keys 17 addends that are cut off at the largest one's bits. Numerator and
    denominator each. `v_scale` as a number: below 2^-22 of the maximum's a FixedI8 cache's weight ends at f16's last bit: 2^-33 of the total."""
    steps = 8 * top * np.log(2) + 16 + weight_steps + 64 + 2.125 * n
    far = 0 if v_scale is None else 2.0 ** -33 * v_scale * np.abs(v.astype(np.float64)).sum(0).repeat(len(mean) // v.shape[1], axis=0)
    return 2 * steps[:, None] * 2.0 ** -24 * mean + far


def _check(got, want, bound):
    low, high = _bf16(want - bound), _bf16(want + bound)
    assert ((low <= got) & (got <= high)).all(), np.maximum(low - got, got - high).max()


def _decode(stream, kern, scaled, q, q_scale, pages, scales, table, lens, sk, sv, temp, window):
    rows, (H, D) = q.shape[0], sk.shape
    out, l = torch.zeros((rows, H * D), dtype=torch.bfloat16, device="cuda"), torch.zeros((rows, H), device="cuda")
    t = [_gpu(a) for a in (q, pages, table, np.array(lens, dtype=np.int32), sk, sv, temp)]
    t_qs, t_s = _gpu(q_scale), _gpu(scales)
    torch.cuda.synchronize()
    if scaled:
        kern.decode_scaled(stream, t[0], t_qs, t[1], t_s, *t[2:], out, l, window)
    else:
        kern.decode(stream, *t, out, l, window)
    stream.synchronize()
    return out.double().cpu().numpy().reshape(rows, H, D), l.cpu().numpy()


@pytest.mark.parametrize("H,Hk,D,page,lens,new,window", [
    (4, 4, 128, 16, [0, 1, 17, 64, 300], 1, 0),
    (4, 2, 64, 32, [1, 40, 200], 2, 48),
    (8, 1, 32, 16, [5, 33, 129], 1, 0),
    (16, 1, 128, 64, [20, 90], 1, 0),
    (24, 1, 64, 16, [31, 160], 1, 0),
    (20, 1, 32, 16, [64], 1, 0),
])
@pytest.mark.parametrize("room", [0, 300000])
def test_bf16_output_is_the_exact_values_but_for_near_ties(stream, H, Hk, D, page, lens, new, window, room):
    rng = np.random.default_rng([5, H, D])
    ends = [n + new - 1 for n in lens]
    table, n_pages = _table(rng, page, ends, room=room)
    pages, scales, seqs = _cache(rng, table, n_pages, Hk, page, D, False, ends)
    q, sk, sv = _codes(rng, len(lens) * new, H * D), _codes(rng, H, D), _codes(rng, H, D, std=1.3)
    temp, q_scale = (0.3 + rng.random(H)).astype(np.float32), np.full((len(q), H), 0.125, dtype=np.float32)
    kern = _kernel(H, Hk, D, page)
    got, _ = _decode(stream, kern, False, q, q_scale, pages, scales, table, lens, sk, sv, temp, window)
    for row in range(len(q)):
        n, (k, ks, v, vs) = lens[row // new] + row % new, seqs[row // new]
        want, _, mean, top = o_paged.attend(q[row].reshape(H, D), q_scale[row], k[:n], ks[:n], v[:n], vs[:n], sk, sv, temp, window)
        _check(got[row], want, _bound(n, top, mean, v[:n], 0.125, 4))


# (what the value scales are like)
SCALES = ["one_far_above", "two_far_above", "wide", "negative"]


@pytest.mark.parametrize("H,Hk,D,page,lens,new", [
    (4, 2, 128, 16, [1, 17, 300], 1),
    (6, 2, 64, 32, [40, 200], 3),
    (8, 1, 32, 16, [33, 129], 2),
    (20, 1, 128, 64, [90], 1),
    (24, 1, 64, 16, [31, 160], 1),
])
@pytest.mark.parametrize("kind", SCALES)
@pytest.mark.parametrize("room", [0, 300000])
def test_value_scales_of_any_size(stream, kind, H, Hk, D, page, lens, new, room):
    """A value with a scale far above the others' takes no bits from theirs: keys that carry next to no weight have scales of 2^60, or
    of 2^20 and 2^100; scales are spread over 2^80; some are below zero."""
    rng = np.random.default_rng([6, H, D])
    ends = [n + new - 1 for n in lens]
    table, n_pages = _table(rng, page, ends, room=room)
    pages, scales, seqs = _cache(rng, table, n_pages, Hk, page, D, True, ends)
    q, sk, sv = np.abs(_codes(rng, len(lens) * new, H * D)), _codes(rng, H, D), _codes(rng, H, D, std=1.3)
    for i, (k, ks, v, vs) in enumerate(seqs):
        n = len(k)
        if kind.endswith("above"):
            for size, at in zip([60] if kind.startswith("one") else [20, 100], rng.permutation(n)):
                k[at], ks[at], vs[at] = -127, 1.0, 2.0 ** size   # (queries have no negative codes: a score hundreds below the others')
        else:
            vs *= np.exp2(rng.uniform(-40, 40, vs.shape)).astype(np.float32) if kind == "wide" else np.where(rng.random(vs.shape) < 0.7, -1, 1)
        p = np.arange(n)
        where = table[i, p // page], slice(None), p % page
        pages[where], scales[where] = np.concatenate((k, v), axis=-1), np.stack((ks, vs), axis=-1)
    temp, q_scale = (0.3 + rng.random(H)).astype(np.float32), (2.0 ** rng.uniform(-5, -2, (len(q), H))).astype(np.float32)
    got, got_l = _decode(stream, _kernel(H, Hk, D, page), True, q, q_scale, pages, scales, table, lens, sk, sv, temp, 0)
    for row in range(len(q)):
        n, (k, ks, v, vs) = lens[row // new] + row % new, seqs[row // new]
        want, want_l, mean, top = o_paged.attend(q[row].reshape(H, D), q_scale[row], k[:n], ks[:n], v[:n], vs[:n], sk, sv, temp, 0)
        _check(got[row], want, _bound(n, top, mean, v[:n], None, 256))   # a weight's two bf16 numbers: 2^-16
        assert (np.abs(got_l[row] - want_l) <= (16 * top + n + 128) * 2.0 ** -23).all()
