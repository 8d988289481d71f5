"""The paged key-value cache on the GPU against its restatement (oracle/paged.py): appending is exact, attention is held to
bounds that are derived from the number of roundings."""
import numpy as np
import pytest
import torch

from oracle import formats, paged as o_paged

pytestmark = pytest.mark.gpu

BAD_INDEX = 16


def _codes(rng, *shape, std=1.0):
    return formats.quantize_fixedi8(rng.standard_normal(shape) * std)


def _bf16(rng, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(torch.bfloat16)


def _gpu(a):
    return (a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))).cuda()


def _table(rng, page, ends, spare=2, room=0):
    """Pages in no order; -1 behind a sequence's last page, room for `room` tokens at least."""
    need = [-(-e // page) for e in ends]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(ends), max(max(need), 1, room // page)), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, len(order)


def _kernel(H, Hk, D, page, q_extra=0, kv_extra=0, o_extra=0, rotary=0, adjacent=False):
    from x17ai_b200 import kernels as K
    return K.PagedAttnKernel(K.PagedConfig(H, Hk, D, page, H * D + q_extra, 2 * Hk * D + kv_extra, H * D + o_extra, rotary, adjacent))


# ---- append ------------------------------------------------------------------------------------------

APPENDS = [
    # H, Hk, D, page, rotary, adjacent, tokens per sequence, first positions, padding, extra columns, with q, kv_out
    (1, 1, 128, 16, 128, False, [1], [0], 0, 0, True, False),
    (4, 4, 128, 64, 128, False, [1], [1500], 0, 0, True, True),
    (32, 8, 128, 32, 128, True, [1] * 37, list(range(0, 37 * 50, 50)), 3, 0, True, False),
    (5, 5, 64, 16, 64, False, [17, 1, 33], [3, 0, 15], 2, 16, True, True),
    (6, 2, 64, 128, 32, True, [300], [127], 0, 32, True, True),
    (7, 7, 32, 16, 32, False, [5, 64], [60000, 11], 1, 0, True, False),
    (16, 1, 128, 64, 32, False, [129], [64], 0, 0, True, False),
    (3, 3, 128, 1024, 0, False, [40, 2], [1000, 5], 0, 0, True, True),
    (8, 2, 32, 16, 0, True, [16], [16], 5, 0, False, False),
    (12, 4, 128, 32, 96, False, [65], [31], 0, 0, True, False),
    (12, 4, 128, 32, 96, True, [65], [31], 0, 0, False, True),
]


def _append_case(case, scaled, seed=0):
    from x17ai_b200 import kernels as K
    H, Hk, D, page, rotary, adjacent, counts, starts, padding, extra, with_q, kv_out = case
    rng = np.random.default_rng([seed, H, D, page, rotary])
    table, n_pages = _table(rng, page, [s + n for s, n in zip(starts, counts)])
    seqs = np.concatenate([np.full(n, i) for i, n in enumerate(counts)] + [np.full(padding, -1)]).astype(np.int32)
    pos = np.concatenate([s + np.arange(n) for s, n in zip(starts, counts)] + [np.zeros(padding)]).astype(np.int32)
    order = rng.permutation(len(seqs))   # tokens come in no order, padding among them
    seqs, pos = seqs[order], pos[order]
    T = len(seqs)
    kern = _kernel(H, Hk, D, page, extra, extra, 0, rotary, adjacent)
    if scaled:
        q, kv = _bf16(rng, T, H * D + extra, std=3.0), _bf16(rng, T, 2 * Hk * D + extra)
    else:
        q, kv = (torch.from_numpy(rng.integers(-128, 128, s, dtype=np.int8)) for s in ((T, H * D + extra), (T, 2 * Hk * D + extra)))
    rope = o_paged.rope_table(int(pos.max()) + 1, rotary) if rotary else None
    return kern, table, n_pages, seqs, pos, q if with_q else None, kv, rope


@pytest.mark.parametrize("case", APPENDS)
def test_append_is_exact(stream, case):
    H, Hk, D, page, rotary, adjacent, counts, starts, padding, extra, with_q, kv_out = case
    kern, table, n_pages, seqs, pos, q, kv, rope = _append_case(case, False)
    T = len(seqs)
    pages = np.random.default_rng(1).integers(-128, 128, (n_pages, Hk, page, 2 * D), dtype=np.int8)
    t_pages = _gpu(pages)
    q_out = torch.full((T, H * D + extra), 99, dtype=torch.int8, device="cuda") if with_q else None
    kvo = torch.full((T, 2 * Hk * D + extra), 99, dtype=torch.int8, device="cuda") if kv_out else None
    args = [None if a is None else _gpu(a) for a in (q, kv, seqs, pos, table)]
    t_rope = None if rope is None else _gpu(rope)
    torch.cuda.synchronize()
    kern.append(stream, *args, t_pages, q_out, t_rope, kvo)
    stream.synchronize()

    real = seqs >= 0
    cs = rope[pos] if rotary else None
    x = kv.numpy()[:, :2 * Hk * D].reshape(T, Hk, 2, D)
    k = o_paged.rotate(np.ascontiguousarray(x[:, :, 0]), cs, rotary, adjacent)
    stored = np.concatenate((k, x[:, :, 1]), axis=-1)
    pages[table[seqs[real], pos[real] // page], :, pos[real] % page] = stored[real]
    assert np.array_equal(t_pages.cpu().numpy(), pages)
    if with_q:
        want = np.full((T, H * D + extra), 99, dtype=np.int8)
        want[real, :H * D] = o_paged.rotate(q.numpy()[:, :H * D].reshape(T, H, D).copy(), cs, rotary, adjacent).reshape(T, H * D)[real]
        assert np.array_equal(q_out.cpu().numpy(), want)
    if kv_out:
        want = np.full((T, 2 * Hk * D + extra), 99, dtype=np.int8)
        want[real, :2 * Hk * D] = stored.reshape(T, 2 * Hk * D)[real]
        assert np.array_equal(kvo.cpu().numpy(), want)


@pytest.mark.parametrize("case", APPENDS)
def test_append_scaled_is_exact(stream, case):
    """Codes and scales are defined in f32 operations: the kernel's are the restatement's bit for bit. Values of heads that are
    zero, tiny or wide are among the inputs."""
    H, Hk, D, page, rotary, adjacent, counts, starts, padding, extra, with_q, _ = case
    kern, table, n_pages, seqs, pos, q, kv, rope = _append_case(case, True)
    T = len(seqs)
    kv[0, :D] = 0                                   # a key of zeros
    kv[0, D:2 * D] *= 2.0 ** -110                   # a value below what a scale is given for
    kv[-1, :D] *= 2.0 ** 60
    pages = np.random.default_rng(1).integers(-128, 128, (n_pages, Hk, page, 2 * D), dtype=np.int8)
    scales = np.random.default_rng(2).random((n_pages, Hk, page, 2), dtype=np.float32)
    t_pages, t_scales = _gpu(pages), _gpu(scales)
    q_out = torch.full((T, H * D + extra), 99, dtype=torch.int8, device="cuda") if with_q else None
    q_scale = torch.full((T, H), 99.0, device="cuda") if with_q else None
    args = [None if a is None else _gpu(a) for a in (q, kv, seqs, pos, table)]
    t_rope = None if rope is None else _gpu(rope)
    torch.cuda.synchronize()
    kern.append_scaled(stream, *args, t_pages, t_scales, q_out, q_scale, t_rope)
    stream.synchronize()

    real = seqs >= 0
    cs = rope[pos] if rotary else None
    x = kv.float().numpy()[:, :2 * Hk * D].reshape(T, Hk, 2, D)
    x = np.stack((o_paged.rotate(np.ascontiguousarray(x[:, :, 0]), cs, rotary, adjacent), x[:, :, 1]), axis=2)
    codes, s = o_paged.quantise(x)
    at = table[seqs[real], pos[real] // page], slice(None), pos[real] % page
    pages[at], scales[at] = codes.reshape(T, Hk, 2 * D)[real], s[real]
    assert np.array_equal(t_scales.cpu().numpy(), scales)
    assert np.array_equal(t_pages.cpu().numpy(), pages)
    # and the codes stand for the values: half a step, and the two roundings of x * (127 / absmax)
    assert (np.abs(codes * s[..., None].astype(np.float64) - x) <= s[..., None] * (0.5 + 3 * 127 * 2.0 ** -24) + 2.0 ** -100).all()
    if with_q:
        codes, s = o_paged.quantise(o_paged.rotate(q.float().numpy()[:, :H * D].reshape(T, H, D).copy(), cs, rotary, adjacent))
        want, want_s = np.full((T, H * D + extra), 99, dtype=np.int8), np.full((T, H), 99.0, dtype=np.float32)
        want[real, :H * D], want_s[real] = codes.reshape(T, H * D)[real], s[real]
        assert np.array_equal(q_out.cpu().numpy(), want) and np.array_equal(q_scale.cpu().numpy(), want_s)


@pytest.mark.parametrize("scaled", [False, True])
def test_append_leaves_out_bad_indexes(scaled):
    """Sequences, positions and pages out of range: the token is not stored, the others are, the status words say so."""
    from x17ai_b200 import device
    stream = device.CudaStream(0)
    H, Hk, D, page = 2, 2, 64, 16
    kern = _kernel(H, Hk, D, page, rotary=64)
    table = np.array([[0, 1], [7, -5], [2, 3]], dtype=np.int32)     # the pool has four pages
    seqs = np.array([0, 3, 1, 1, 0, 0, 2, 2, 0], dtype=np.int32)
    pos = np.array([5, 0, 3, 20, 32, -1, 31, 2 ** 31 - 1, 30], dtype=np.int32)
    rng = np.random.default_rng(3)
    T = len(seqs)
    q, kv = (_bf16(rng, T, H * D), _bf16(rng, T, 2 * Hk * D)) if scaled else (_codes(rng, T, H * D), _codes(rng, T, 2 * Hk * D))
    pages = torch.full((4, Hk, page, 2 * D), 77, dtype=torch.int8, device="cuda")
    q_out = torch.full((T, H * D), 99, dtype=torch.int8, device="cuda")
    rope = np.concatenate((o_paged.rope_table(30, 64), o_paged.rope_table(32, 64)[30:]))
    for rows, ok in ((30, [0]), (32, [0, 6, 8])):   # positions 30 and 31 lie behind the shorter table
        args = [_gpu(a) for a in (q, kv, seqs, pos, table)]
        t_rope = _gpu(rope[:rows])
        pages.fill_(77)
        q_out.fill_(99)
        extra = (kern.page_scales(4), q_out, torch.zeros((T, H), device="cuda")) if scaled else (q_out,)
        torch.cuda.synchronize()
        (kern.append_scaled if scaled else kern.append)(stream, *args, pages, *extra, t_rope)
        stream.synchronize()
        status = stream.read_status()
        assert status[0] >> 16 == BAD_INDEX and status[2] > 0
        changed = sorted({(a, c) for a, _, c, _ in (pages != 77).nonzero().tolist()})
        assert changed == sorted((int(table[seqs[i], pos[i] // page]), int(pos[i] % page)) for i in ok)
        assert [i for i in range(T) if (q_out[i] != 99).any()] == ok
    assert stream.read_status() == [0, 0, 0, 0]
    stream.close()


# ---- decode ------------------------------------------------------------------------------------------

def _cache(rng, table, n_pages, Hk, page, D, scaled, ends):
    """(pages, scales) full of other data, and per sequence (k, k_scale, v, v_scale) of its keys."""
    pages = rng.integers(-128, 128, (n_pages, Hk, page, 2 * D), dtype=np.int8)
    scales = np.full((n_pages, Hk, page, 2), np.nan, dtype=np.float32)
    scales[::2] = np.inf
    seqs = []
    for i, n in enumerate(ends):
        k, v = _codes(rng, n, Hk, D), _codes(rng, n, Hk, D, std=1.3)
        ks, vs = (np.full((n, Hk), 0.125, dtype=np.float32) for _ in range(2))
        if scaled:
            ks, vs = ((2.0 ** rng.uniform(-6, -1, (n, Hk))).astype(np.float32) for _ in range(2))
        p = np.arange(n)
        where = table[i, p // page], slice(None), p % page
        pages[where] = np.concatenate((k, v), axis=-1)
        scales[where] = np.stack((ks, vs), axis=-1)
        seqs.append((k, ks, v, vs))
    return pages, scales, seqs


def _decode_bounds(n, top, mean, v, v_scale, fixed):
    """Absolute bounds of (value, l). A score carries eight roundings of 2^-24 (temperature, scales, products), a probability
    16 steps of 2^-24 more (exponential, 22 bits kept), a sum over n keys in any order at most n / 4 + 64 in a chain of four
    partial sums or more; numerator and denominator each have them. A weight's low part is rounded to f16, whose smallest step is
    2^-24: half of it, in units of 2^(m - 8) for a score m that is in the total, is at most 2^-33 of the total, and it multiplies
    |code| times a unit no larger than twice the largest v_scale: with a weight of 2^-60 the value is gone. For bf16 output a
    weight has no low part: half a step of f16, 2^-11 of the weight."""
    rel = (8 * top * np.log(2) + 16 + n / 4 + 64) * 2.0 ** -24
    heads = len(mean)
    far = 2.0 ** -32 * (v_scale.max(initial=0) * np.abs(v.astype(np.float64)).sum(0)).repeat(heads // v.shape[1], axis=0)
    return (2 * rel + (0 if fixed else 2.0 ** -11)) * mean + far, rel / np.log(2) + 8 * 2.0 ** -24 * (top + 8 + np.log2(n + 1))


def _check_decode(got, got_l, want, want_l, bound, bound_l, fixed):
    if fixed:   # the code nearest to 8 times a value that is off by at most `bound`
        assert (np.abs(got - np.clip(8 * want, -127, 127)) <= 0.5 + 8 * bound).all()
    else:       # bf16: half a step is 2^-8 of the value
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 1.01 * bound).all(), np.abs(got - want).max()
    if got_l is not None:
        assert (np.abs(got_l - want_l) <= bound_l).all(), (np.abs(got_l - want_l) / bound_l).max()


def _run_decode(stream, H, Hk, D, page, lens, new, window, scaled, fixed, own_scratch=False, extra=0, seed=0, with_l=True, room=0):
    rng = np.random.default_rng([seed, H, D, page, new, len(lens)])
    ends = [n + new - 1 for n in lens]
    table, n_pages = _table(rng, page, ends, room=room)
    pages, scales, seqs = _cache(rng, table, n_pages, Hk, page, D, scaled, ends)
    B = len(lens)
    q = _codes(rng, B * new, H * D + extra)
    q_scale = (2.0 ** rng.uniform(-5, -2, (B * new, H))).astype(np.float32) if scaled else np.full((B * new, H), 0.125, dtype=np.float32)
    sk, sv = _codes(rng, H, D), _codes(rng, H, D, std=1.3)
    temp = (0.3 + rng.random(H)).astype(np.float32)
    kern = _kernel(H, Hk, D, page, extra, 0, extra)
    out = torch.full((B * new, H * D + extra), 55, dtype=torch.int8 if fixed else torch.bfloat16, device="cuda")
    l = torch.full((B * new, H), -7.0, device="cuda") if with_l else None
    t = [_gpu(a) for a in (q, pages, table, np.array(lens, dtype=np.int32), sk, sv, temp)]
    t_qs, t_s = _gpu(q_scale), _gpu(scales)
    scratch = kern.scratch(stream, B, new).fill_(255) if own_scratch else None   # (what it holds is of no account)
    torch.cuda.synchronize()
    if scaled:
        kern.decode_scaled(stream, t[0], t_qs, t[1], t_s, *t[2:], out, l, window, scratch)
    else:
        kern.decode(stream, *t, out, l, window, scratch)
    stream.synchronize()
    got, got_l = out.float().cpu().numpy(), l.cpu().numpy() if with_l else None
    assert (got[:, H * D:] == 55).all()
    for b in range(B):
        k, ks, v, vs = seqs[b]
        for i in range(new):
            row, n = b * new + i, lens[b] + i
            want, want_l, mean, top = o_paged.attend(q[row, :H * D].reshape(H, D), q_scale[row], k[:n], ks[:n], v[:n], vs[:n], sk, sv, temp,
                                                     window)
            bound, bound_l = _decode_bounds(n, top[:, None], mean, v[:n], vs[:n], fixed)
            _check_decode(got[row, :H * D].reshape(H, D), None if got_l is None else got_l[row], want, want_l, bound, bound_l[:, 0], fixed)


DECODES = [
    # H, Hk, D, page, lens, new, window
    (1, 1, 128, 16, [1], 1, 0),
    (4, 4, 128, 16, [0, 1, 15, 16, 17, 300], 1, 0),
    (4, 4, 64, 64, [0, 1, 31, 32, 33, 500], 1, 0),
    (4, 4, 32, 32, [0, 1, 63, 64, 65, 700], 1, 0),
    (8, 1, 128, 32, [1000, 3], 1, 0),
    (6, 2, 64, 128, [129, 1], 1, 0),
    (20, 4, 128, 64, [777], 1, 0),
    (16, 1, 64, 16, [90, 2000], 1, 0),
    (17, 1, 32, 16, [45], 1, 0),
    (9, 3, 128, 1024, [2050, 1023], 1, 0),
    (4, 2, 128, 16, [0, 5, 16, 17, 400], 1, 16),
    (4, 2, 64, 32, [39, 40, 512, 600], 1, 48),
    (4, 4, 32, 64, [1000], 1, 512),
    (2, 2, 128, 16, [0, 1, 14, 200], 2, 0),
    (3, 3, 64, 32, [0, 30, 300], 5, 32),
    (16, 2, 128, 64, [0, 60, 127], 7, 0),
    (7, 7, 32, 16, [15, 16], 9, 0),
    (4, 4, 64, 16, [100], 64, 64),
]


@pytest.mark.parametrize("H,Hk,D,page,lens,new,window", DECODES)
@pytest.mark.parametrize("kind", ["bf16", "fixed", "scaled"])
@pytest.mark.parametrize("room", [0, 300000])
def test_decode(stream, kind, H, Hk, D, page, lens, new, window, room):
    """With room for few keys a sequence has CTAs of its own, with room for many all sequences share the chip's (a window
    counts as room)."""
    _run_decode(stream, H, Hk, D, page, lens, new, window, kind == "scaled", kind == "fixed", room=room)


@pytest.mark.parametrize("kind", ["bf16", "fixed", "scaled"])
@pytest.mark.parametrize("own_scratch", [False, True])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_decode_long(stream, kind, D, own_scratch):
    """Sequences that many warps share, wider rows than the heads need, no L."""
    _run_decode(stream, 8, 2, D, 64, [5000, 9001], 1, 0, kind == "scaled", kind == "fixed", own_scratch, extra=16, with_l=False)


@pytest.mark.parametrize("kind", ["bf16", "fixed", "scaled"])
def test_decode_many_sequences(stream, kind):
    """More (sequence, key head) pairs than warps: a warp goes through several, parts of the first and the last of them; more
    than 32 sequences, some of them empty."""
    _run_decode(stream, 16, 16, 64, 16, [(37 * i) % 301 for i in range(150)], 1, 0, kind == "scaled", kind == "fixed")
    _run_decode(stream, 24, 8, 32, 32, [(91 * i) % 777 for i in range(70)], 3, 64, kind == "scaled", kind == "fixed", seed=1)


@pytest.mark.parametrize("H,Hk,D,page,lens,new,window", [
    (20, 1, 128, 64, [0, 1, 33, 2100], 1, 0),
    (6, 2, 128, 16, [0, 40, 700], 7, 48),
    (24, 1, 64, 32, [5, 3000], 1, 0),
    (14, 2, 64, 16, [0, 63, 64, 900], 3, 0),
    (17, 1, 32, 128, [1, 130, 2500], 1, 0),
    (8, 1, 32, 16, [0, 200, 201], 3, 128),
    (25, 1, 64, 16, [300, 0], 1, 0),
])
@pytest.mark.parametrize("kind", ["bf16", "fixed", "scaled"])
@pytest.mark.parametrize("room", [0, 300000])
def test_decode_rows_of_three_tiles(stream, kind, H, Hk, D, page, lens, new, window, room):
    """17 to 24 rows of a key head, and one more."""
    _run_decode(stream, H, Hk, D, page, lens, new, window, kind == "scaled", kind == "fixed", room=room)


@pytest.mark.parametrize("kind", ["bf16", "fixed", "scaled"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_decode_rows_of_three_tiles_many_sequences(stream, kind, D):
    _run_decode(stream, 36, 6, D, 32, [(53 * i) % 700 for i in range(70)], 4, 0, kind == "scaled", kind == "fixed", seed=3)


def test_scratch_that_is_too_small(stream):
    from x17ai_b200 import X17Error
    H, D, page = 4, 64, 16
    kern = _kernel(H, H, D, page)
    z = lambda dtype, *shape: torch.zeros(shape, dtype=dtype, device="cuda")
    args = (z(torch.int8, 2, H * D), kern.pages(4), z(torch.int32, 2, 20000), z(torch.int32, 2), z(torch.int8, H, D), z(torch.int8, H, D),
            z(torch.float32, H), z(torch.bfloat16, 2, H * D))
    scratch = kern.scratch(stream, 2)
    torch.cuda.synchronize()
    kern.decode(stream, *args, scratch=scratch)
    with pytest.raises(X17Error, match="scratch must be 16-byte aligned and have"):
        kern.decode(stream, *args, scratch=scratch[:-1])
    with pytest.raises(X17Error, match="scratch must be 16-byte aligned and have"):
        kern.decode(stream, *args, scratch=torch.cat((scratch, scratch))[8:])
    with pytest.raises(X17Error, match="64 new tokens"):
        kern.scratch(stream, 2, 65)


def test_decode_scores_far_apart(stream):
    """Scores that differ by hundreds: one key carries all the weight, wherever it lies; and a sink above every key."""
    H = Hk = 2
    D, page, n = 128, 16, 700
    rng = np.random.default_rng(1)
    table, n_pages = _table(rng, page, [n])
    pages, scales, seqs = _cache(rng, table, n_pages, Hk, page, D, False, [n])
    q = np.full((1, H * D), 127, dtype=np.int8)
    sv = _codes(rng, H, D)
    for at in (0, 5, 350, 699, None):
        sk = np.full((H, D), 0 if at is not None else 127, dtype=np.int8)
        if at is not None:
            pages[table[0, at // page], :, at % page, :D] = 127
        kern = _kernel(H, Hk, D, page)
        out, l = torch.zeros((1, H * D), dtype=torch.int8, device="cuda"), torch.zeros((1, H), device="cuda")
        temp = np.full(H, 4.0, dtype=np.float32)
        t = [_gpu(a) for a in (q, pages, table, np.array([n], dtype=np.int32), sk, sv, temp)]
        torch.cuda.synchronize()
        kern.decode(stream, *t, out, l)
        stream.synchronize()
        want = sv if at is None else pages[table[0, at // page], :, at % page, D:]
        assert np.array_equal(out.cpu().numpy().reshape(H, D), np.clip(want, -127, 127))
        assert np.allclose(l.cpu().numpy(), np.log2(255) + 127 * 127 / 64 * D ** 0.5 * 4 * np.log2(n + 4), rtol=1e-6)
        if at is not None:   # put the key back
            pages[table[0, at // page], :, at % page, :D] = seqs[0][0][at]


def test_decode_lengths_beyond_the_table(stream):
    """Lengths above the table's capacity are clamped to it, negative ones to 0."""
    H = Hk = 2
    D, page = 64, 16
    rng = np.random.default_rng(4)
    table, n_pages = _table(rng, page, [64, 64, 64], spare=0)
    pages = _codes(rng, n_pages, Hk, page, 2 * D)
    q, sk, sv, temp = _codes(rng, 3, H * D), _codes(rng, H, D), _codes(rng, H, D), np.ones(H, dtype=np.float32)
    kern, outs = _kernel(H, Hk, D, page), []
    for lens in ([5000, -3, 2 ** 31 - 1], [64, 0, 64]):
        out = torch.zeros((3, H * D), dtype=torch.bfloat16, device="cuda")
        t = [_gpu(a) for a in (q, pages, table, np.array(lens, dtype=np.int32), sk, sv, temp)]
        torch.cuda.synchronize()
        kern.decode(stream, *t, out)
        stream.synchronize()
        outs.append(out)
    assert outs[0].any() and torch.equal(*outs)


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("room", [0, 300000])
def test_decode_leaves_out_bad_pages(scaled, room):
    """A key on a page outside the pool is not attended to; the status words say so."""
    from x17ai_b200 import device
    stream = device.CudaStream(0)
    H, Hk, D, page, n = 4, 2, 64, 16, 100
    rng = np.random.default_rng(6)
    table, n_pages = _table(rng, page, [n, n], room=room)
    pages, scales, seqs = _cache(rng, table, n_pages, Hk, page, D, scaled, [n, n])
    table[0, 2], table[0, 6], table[1, 0] = n_pages, -1, 2 ** 31 - 1
    keep = [np.r_[0:32, 48:96], np.r_[16:100]]
    q, sk, sv, temp = _codes(rng, 2, H * D), _codes(rng, H, D), _codes(rng, H, D), np.ones(H, dtype=np.float32)
    q_scale = np.full((2, H), 0.125, dtype=np.float32)
    kern = _kernel(H, Hk, D, page)
    out, l = torch.zeros((2, H * D), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, H), device="cuda")
    t = [_gpu(a) for a in (q, pages, table, np.array([n, n], dtype=np.int32), sk, sv, temp)]
    t_qs, t_s = _gpu(q_scale), _gpu(scales)
    torch.cuda.synchronize()
    if scaled:
        kern.decode_scaled(stream, t[0], t_qs, t[1], t_s, *t[2:], out, l)
    else:
        kern.decode(stream, *t, out, l)
    stream.synchronize()
    status = stream.read_status()
    assert status[0] >> 16 == BAD_INDEX and status[2] > 0
    stream.close()
    for b in range(2):
        k, ks, v, vs = (a[keep[b]] for a in seqs[b])
        # the temperature goes by the length, not by the keys that are left
        fix = np.float32(np.log2(n + 4) / np.log2(len(k) + 4))
        want, want_l, mean, top = o_paged.attend(q[b].reshape(H, D), q_scale[b], k, ks, v, vs, sk, sv, temp * fix, 0)
        bound, bound_l = _decode_bounds(n, top[:, None], mean, v, vs, False)
        _check_decode(out[b].float().cpu().numpy().reshape(H, D), l[b].cpu().numpy(), want, want_l, bound + 1e-6 * mean, bound_l[:, 0] + 1e-5,
                      False)


def test_offsets_beyond_32_bits(stream):
    """A pool of 5 GB whose last pages are in use: append and decode reach them."""
    H, Hk, D, page = 8, 8, 128, 128
    n_pages = 5 * 2 ** 30 // (Hk * page * 2 * D)
    pages = torch.zeros((n_pages, Hk, page, 2 * D), dtype=torch.int8, device="cuda")
    table = np.array([[n_pages - 1, n_pages - 3]], dtype=np.int32)
    rng = np.random.default_rng(8)
    n = 200
    kv, q = _codes(rng, n, 2 * Hk * D), _codes(rng, 1, H * D)
    sk, sv, temp = _codes(rng, H, D), _codes(rng, H, D), np.ones(H, dtype=np.float32)
    kern = _kernel(H, Hk, D, page)
    out, l = torch.zeros((1, H * D), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, H), device="cuda")
    t = [_gpu(a) for a in (kv, np.zeros(n, dtype=np.int32), np.arange(n, dtype=np.int32), table)]
    rest = [_gpu(a) for a in (np.array([n], dtype=np.int32), sk, sv, temp)]
    t_q = _gpu(q)
    torch.cuda.synchronize()
    kern.append(stream, None, *t, pages, None)
    kern.decode(stream, t_q, pages, t[3], *rest, out, l)
    stream.synchronize()
    x = kv.reshape(n, Hk, 2, D)
    assert np.array_equal(pages[n_pages - 1].cpu().numpy(), x[:128].transpose(1, 0, 2, 3).reshape(Hk, 128, 2 * D))
    assert not pages[n_pages - 2].any() and not pages[:n_pages - 3].any()
    eighth = np.full((n, Hk), 0.125)
    want, want_l, mean, top = o_paged.attend(q.reshape(H, D), np.full(H, 0.125), x[:, :, 0], eighth, x[:, :, 1], eighth, sk, sv, temp, 0)
    bound, bound_l = _decode_bounds(n, top[:, None], mean, x[:, :, 1], eighth, False)
    _check_decode(out.float().cpu().numpy().reshape(H, D), l[0].cpu().numpy(), want, want_l, bound, bound_l[:, 0], False)


# ---- together, as they are used ------------------------------------------------------------------------

def _served(stream, steps=4):
    """A batch through prompt and decode steps: projections, append, decode, output projection. Yields what each step gave."""
    from x17ai_b200 import kernels as K
    B, H, D, dm, page, prompt = 3, 4, 64, 256, 16, 37
    rng = np.random.default_rng(11)
    w_q, w_kv, w_o = (_gpu(_codes(rng, r, c)) for r, c in ((H * D, dm), (2 * H * D, dm), (2 * dm, H * D)))
    k_q, k_kv = K.GemmKernel(K.attn_q_fwd_config(dm, H * D)), K.GemmKernel(K.attn_kv_fwd_config(dm, 2 * H * D, D))
    k_o = K.GemmKernel(K.attn_y_fwd_config(H * D, dm))
    kern = _kernel(H, H, D, page, rotary=D)
    ends = [prompt + i * 5 + steps for i in range(B)]
    table, n_pages = _table(rng, page, ends)
    pages, rope = kern.pages(n_pages), K.rope_table(max(ends), D)
    sk, sv, temp = _gpu(_codes(rng, H, D)), _gpu(_codes(rng, H, D)), _gpu(np.ones(H, dtype=np.float32))
    T = sum(prompt + i * 5 for i in range(B))
    seqs = np.concatenate([np.full(prompt + i * 5, i) for i in range(B)]).astype(np.int32)
    pos = np.concatenate([np.arange(prompt + i * 5) for i in range(B)]).astype(np.int32)
    x = [_gpu(_codes(rng, T, dm))] + [_gpu(_codes(rng, B, dm)) for _ in range(steps)]
    index = [(_gpu(seqs), _gpu(pos))] + [(_gpu(np.arange(B, dtype=np.int32)), _gpu(np.array([e - steps + s for e in ends], dtype=np.int32)))
                                         for s in range(steps)]
    t_table = _gpu(table)
    results = []
    for s, (xs, (sq, ps)) in enumerate(zip(x, index)):
        rows = xs.shape[0]
        new = lambda cols, dtype=torch.int8: torch.zeros((rows, cols), dtype=dtype, device="cuda")
        q, kv, rr, q_out, kv_out, out, y = (new(H * D), new(2 * H * D), new(H, torch.float32), new(H * D), new(2 * H * D), new(H * D),
                                            new(dm, torch.uint8))
        torch.cuda.synchronize()
        k_q.launch(stream, xs, w_q, q)
        k_kv.launch(stream, xs, w_kv, kv, rrms=rr)
        kern.append(stream, q, kv, sq, ps, t_table, pages, q_out, rope, kv_out)
        if s > 0:
            kern.decode(stream, q_out, pages, t_table, ps, sk, sv, temp, out)
            k_o.launch(stream, out, w_o, y, residual=xs)
        results.append((q_out, kv_out, out, y))
    stream.synchronize()
    return kern, (sk, sv, temp), seqs, pos, ends, steps, results


def test_serving_steps(stream):
    """Prompt and decode steps give what the contiguous decode gives on the rotated rows, within a code (its probabilities have
    eight bits)."""
    from x17ai_b200 import kernels as K
    kern, (sk, sv, temp), seqs, pos, ends, steps, results = _served(stream)
    B, H, D = len(ends), 4, 64
    cap = max(ends)
    flat = torch.zeros((B, cap, 2 * H * D), dtype=torch.int8, device="cuda")
    flat[torch.from_numpy(seqs).cuda().long(), torch.from_numpy(pos).cuda().long()] = results[0][1]
    attn = K.AttnKernel(K.AttnKernelConfig(H, D, H * D, 2 * H * D, H * D))
    for s in range(steps):
        q_out, kv_out, out, y = results[1 + s]
        at = torch.tensor([e - steps + s for e in ends], device="cuda")
        flat[torch.arange(B, device="cuda"), at] = kv_out
        want = torch.zeros_like(out)
        lens = at.to(torch.int32)
        torch.cuda.synchronize()
        attn.decode(stream, q_out, flat, cap, sk, sv, temp, want, kv_lens=lens)
        stream.synchronize()
        d = (out.int() - want.int()).abs()
        assert out.any() and y.any() and d.max() <= 1 and (d > 0).float().mean() <= 0.08


def test_drafted_tokens_equal_single_steps(stream):
    """n tokens of a sequence in one call are n calls of one token at growing lengths: the same keys, to the bounds of a
    regrouped sum: two roundings to bf16 of 2^-8, and weights that two different maxima round to f16, 2^-11 each of the largest
    value."""
    H, Hk, D, page, new = 6, 2, 128, 32, 5
    lens = [0, 29, 300]
    rng = np.random.default_rng(21)
    table, n_pages = _table(rng, page, [n + new for n in lens])
    pages, _, seqs = _cache(rng, table, n_pages, Hk, page, D, False, [n + new for n in lens])
    most = max(int(np.abs(v.astype(np.int32)).max()) for _, _, v, _ in seqs) / 8
    q, sk, sv, temp = _codes(rng, len(lens) * new, H * D), _codes(rng, H, D), _codes(rng, H, D), np.ones(H, dtype=np.float32)
    kern = _kernel(H, Hk, D, page)
    t_q, t_pages, t_table, t_sk, t_sv, t_temp = (_gpu(a) for a in (q, pages, table, sk, sv, temp))
    for window in (0, 64):
        out = torch.zeros((len(lens) * new, H * D), dtype=torch.bfloat16, device="cuda")
        l = torch.zeros((len(lens) * new, H), device="cuda")
        t_lens = _gpu(np.array(lens, dtype=np.int32))
        torch.cuda.synchronize()
        kern.decode(stream, t_q, t_pages, t_table, t_lens, t_sk, t_sv, t_temp, out, l, window)
        stream.synchronize()
        for i in range(new):
            one, one_l = torch.zeros((len(lens), H * D), dtype=torch.bfloat16, device="cuda"), torch.zeros((len(lens), H), device="cuda")
            q_i, lens_i = t_q[i::new].contiguous(), t_lens + i
            torch.cuda.synchronize()
            kern.decode(stream, q_i, t_pages, t_table, lens_i, t_sk, t_sv, t_temp, one, one_l, window)
            stream.synchronize()
            assert (out[i::new].float() - one.float()).abs().le(2.0 ** -7 * one.float().abs() + 2.0 ** -10 * most + 1e-4).all()
            assert (l[i::new] - one_l).abs().max() <= 1e-4


@pytest.mark.parametrize("room,kernels", [(0, 2), (300000, 3)])
def test_captured_and_replayed(room, kernels):
    """A step recorded once and replayed with other positions, lengths and rows in the same buffers; two graphs at once on two
    streams, which share the pool and write different pages."""
    from x17ai_b200 import device, kernels as K
    H, Hk, D, page, B = 8, 2, 64, 16, 4
    rng = np.random.default_rng(31)
    table, n_pages = _table(rng, page, [200] * (2 * B), room=room)
    pages, _, _ = _cache(rng, table, n_pages, Hk, page, D, False, [200] * (2 * B))
    t_pages, rope = _gpu(pages), K.rope_table(256, D)
    kern = _kernel(H, Hk, D, page, rotary=D)
    sk, sv, temp = _gpu(_codes(rng, H, D)), _gpu(_codes(rng, H, D)), _gpu(np.ones(H, dtype=np.float32))
    sides = []
    for half in range(2):
        s = device.CudaStream(0)
        x = dict(q=torch.zeros((B, H * D), dtype=torch.int8, device="cuda"), kv=torch.zeros((B, 2 * Hk * D), dtype=torch.int8, device="cuda"),
                 seqs=_gpu(np.arange(B, dtype=np.int32)), pos=torch.zeros(B, dtype=torch.int32, device="cuda"),
                 table=_gpu(table[half * B:half * B + B]), q_out=torch.zeros((B, H * D), dtype=torch.int8, device="cuda"),
                 out=torch.zeros((B, H * D), dtype=torch.bfloat16, device="cuda"))
        torch.cuda.synchronize()

        def step(x=x, s=s):
            kern.append(s, x["q"], x["kv"], x["seqs"], x["pos"], x["table"], t_pages, x["q_out"], rope)
            kern.decode(s, x["q_out"], t_pages, x["table"], x["pos"], sk, sv, temp, x["out"])
        step()
        s.synchronize()
        with device.CudaGraph(s) as g:
            step()
        assert g.kernel_nodes == kernels
        sides.append((s, x, step, g))
    for turn in range(3):
        fresh = [(_gpu(_codes(rng, B, H * D)), _gpu(_codes(rng, B, 2 * Hk * D)), _gpu(rng.integers(0, 199, B).astype(np.int32))) for _ in sides]
        torch.cuda.synchronize()
        wants = []
        for (s, x, step, g), (q, kv, pos) in zip(sides, fresh):
            x["q"].copy_(q), x["kv"].copy_(kv), x["pos"].copy_(pos)
            torch.cuda.synchronize()
            step()
            s.synchronize()
            wants.append(x["out"].clone())
            x["out"].zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for s, x, step, g in sides:
                g.launch()
        for (s, x, step, g), want in zip(sides, wants):
            s.synchronize()
            assert want.any() and torch.equal(x["out"], want)
    for s, x, step, g in sides:
        assert s.read_status() == [0, 0, 0, 0]
        g.destroy()
        s.close()


@pytest.mark.parametrize("room", [0, 300000])
def test_reads_what_torch_wrote_in_front(room):
    """Inputs written by torch on the same stream right in front of the calls, changing from pass to pass, nothing waited for."""
    from x17ai_b200 import device, kernels as K
    H, Hk, D, page, B, n = 8, 2, 128, 32, 5, 24
    rng = np.random.default_rng(41)
    table, n_pages = _table(rng, page, [400] * B, room=room)
    kern, rope = _kernel(H, Hk, D, page, rotary=D), K.rope_table(512, D)
    sk, sv, temp = _gpu(_codes(rng, H, D)), _gpu(_codes(rng, H, D)), _gpu(np.ones(H, dtype=np.float32))
    src = [(_gpu(_codes(rng, n_pages, Hk, page, 2 * D)), _gpu(_codes(rng, B, H * D)), _gpu(_codes(rng, B, 2 * Hk * D)),
            _gpu(rng.integers(0, 399, B).astype(np.int32)), _gpu(table[rng.permutation(B)])) for _ in range(3)]
    pages, q, kv, pos, t_table = (torch.zeros_like(t) for t in src[0])
    seqs, q_out = _gpu(np.arange(B, dtype=np.int32)), torch.zeros((B, H * D), dtype=torch.int8, device="cuda")
    outs = torch.zeros((n, B, H * D), dtype=torch.bfloat16, device="cuda")
    want = torch.zeros((3, B, H * D), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        st = device.TorchStream()

        def go(i, out, wait):
            for dst, x in zip((pages, q, kv, pos, t_table), src[i]):
                dst.copy_(x)
            if wait:
                side.synchronize()
            kern.append(st, q, kv, seqs, pos, t_table, pages, q_out, rope)
            if wait:
                side.synchronize()
            kern.decode(st, q_out, pages, t_table, pos, sk, sv, temp, out)
            if wait:
                side.synchronize()
        for i in range(3):
            go(i, want[i], True)
        for i in range(n):
            go(i % 3, outs[i], False)
    side.synchronize()
    assert st.read_status() == [0, 0, 0, 0]
    assert want.any() and all(torch.equal(outs[i], want[i % 3]) for i in range(n))


@pytest.mark.parametrize("kind", ["bf16", "fixed", "scaled"])
@pytest.mark.parametrize("H,Hk", [(8, 8), (80, 8)])
def test_decode_more_work_than_the_chip_holds(stream, kind, H, Hk):
    """More than 30 steps for every warp, so that more CTAs than the chip holds at once share the list. All sequences name the same
    pages, each up to a length of its own. Twice, with the same bits."""
    D, page, B, cap, scaled, fixed = 128, 64, 66, 3712, kind == "scaled", kind == "fixed"
    rng = np.random.default_rng([71, H])
    ends = [int(n) for n in rng.integers(3300, cap + 1, B)]
    ends[7], ends[40] = 0, 1
    one, n_pages = _table(rng, page, [cap])
    pages, scales, ((k, ks, v, vs),) = _cache(rng, one, n_pages, Hk, page, D, scaled, [cap])
    q = _codes(rng, B, H * D)
    q_scale = (2.0 ** rng.uniform(-5, -2, (B, H))).astype(np.float32) if scaled else np.full((B, H), 0.125, dtype=np.float32)
    sk, sv, temp = _codes(rng, H, D), _codes(rng, H, D, std=1.3), (0.3 + rng.random(H)).astype(np.float32)
    kern = _kernel(H, Hk, D, page)
    t = [_gpu(a) for a in (q, pages, np.repeat(one, B, axis=0), np.array(ends, dtype=np.int32), sk, sv, temp)]
    t_qs, t_s = _gpu(q_scale), _gpu(scales)
    results = []
    for _ in range(2):
        out, l = torch.zeros((B, H * D), dtype=torch.int8 if fixed else torch.bfloat16, device="cuda"), torch.zeros((B, H), device="cuda")
        torch.cuda.synchronize()
        if scaled:
            kern.decode_scaled(stream, t[0], t_qs, t[1], t_s, *t[2:], out, l)
        else:
            kern.decode(stream, *t, out, l)
        stream.synchronize()
        results.append((out, l))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    got, got_l = results[0][0].float().cpu().numpy(), results[0][1].cpu().numpy()
    for b in (0, 1, 6, 7, 8, 31, 32, 39, 40, 41, 64, 65):
        n = ends[b]
        want, want_l, mean, top = o_paged.attend(q[b].reshape(H, D), q_scale[b], k[:n], ks[:n], v[:n], vs[:n], sk, sv, temp, 0)
        bound, bound_l = _decode_bounds(n, top[:, None], mean, v[:n], vs[:n], fixed)
        _check_decode(got[b].reshape(H, D), got_l[b], want, want_l, bound, bound_l[:, 0], fixed)


@pytest.mark.parametrize("kind", ["fixed", "scaled"])
@pytest.mark.parametrize("room", [0, 300000])
def test_decode_most_rows(stream, kind, room):
    """64 query heads of one key head, 64 new tokens: 4096 rows, 256 chunks of them."""
    _run_decode(stream, 64, 1, 32, 32, [70], 64, 32, kind == "scaled", kind == "fixed", room=room)


def test_append_and_decode_at_the_same_time(stream):
    """Two sequences of calls on two streams, not captured, without scratch memory of their own: what each writes is its own."""
    from x17ai_b200 import device, kernels as K
    H, Hk, D, page, B = 8, 2, 128, 16, 3
    rng = np.random.default_rng(51)
    table, n_pages = _table(rng, page, [900] * (2 * B), room=300000)
    pages, _, _ = _cache(rng, table, n_pages, Hk, page, D, False, [900] * (2 * B))
    kern, rope, t_pages = _kernel(H, Hk, D, page, rotary=D), K.rope_table(1024, D), _gpu(pages)
    sk, sv, temp = _gpu(_codes(rng, H, D)), _gpu(_codes(rng, H, D)), _gpu(np.ones(H, dtype=np.float32))
    streams = [stream, device.CudaStream(0)]
    n = 40
    sides = [dict(q=_gpu(_codes(rng, n, B, H * D)), kv=_gpu(_codes(rng, n, B, 2 * Hk * D)), seqs=_gpu(np.arange(B, dtype=np.int32)),
                  pos=_gpu((np.arange(n)[:, None] + rng.integers(0, 850, B)).astype(np.int32)), table=_gpu(table[i * B:i * B + B]),
                  q_out=torch.zeros((n, B, H * D), dtype=torch.int8, device="cuda")) for i in range(2)]

    def go(s, x, i, out):
        kern.append(s, x["q"][i], x["kv"][i], x["seqs"], x["pos"][i], x["table"], t_pages, x["q_out"][i], rope)
        kern.decode(s, x["q_out"][i], t_pages, x["table"], x["pos"][i], sk, sv, temp, out[i])
    start = t_pages.clone()
    outs = []
    for together in (False, True):
        t_pages.copy_(start)
        o = [torch.zeros((n, B, H * D), dtype=torch.bfloat16, device="cuda") for _ in sides]
        torch.cuda.synchronize()
        for i in range(n):
            for s, x, out in zip(streams, sides, o):
                go(s, x, i, out)
                if not together:
                    s.synchronize()
        torch.cuda.synchronize()
        outs.append((o, t_pages.clone()))
    assert torch.equal(outs[0][1], outs[1][1])
    for a, b in zip(outs[0][0], outs[1][0]):
        assert a.any() and torch.equal(a, b)
    streams[1].close()


FIRST_IN_A_CAPTURE = """
import torch
from x17ai_b200 import device, kernels as K
H, D, page = 2, 64, 16
kern = K.PagedAttnKernel(K.PagedConfig(H, H, D, page, H * D, 2 * H * D, H * D))
s = device.CudaStream(0)
gen = torch.Generator(device="cuda").manual_seed(1)
codes = lambda *shape: torch.randint(-20, 21, shape, dtype=torch.int8, device="cuda", generator=gen)
pages, q, sk, sv = codes(8, H, page, 2 * D), codes(1, H * D), codes(H, D), codes(H, D)
table = torch.zeros((1, 20000), dtype=torch.int32, device="cuda")
table[0, :8] = torch.arange(8, device="cuda")
lens, temp = torch.full((1,), 100, dtype=torch.int32, device="cuda"), torch.ones(H, device="cuda")
out, again, narrow = (torch.zeros((1, H * D), dtype=torch.bfloat16, device="cuda") for _ in range(3))
narrow_table = table[:, :200].contiguous()
torch.cuda.synchronize()
with device.CudaGraph(s) as g:
    kern.decode(s, q, pages, narrow_table, lens, sk, sv, temp, narrow)
    kern.decode(s, q, pages, table, lens, sk, sv, temp, out)
assert g.kernel_nodes == 3   # a cluster for every key head; the list and what joins its parts
for _ in range(3):
    g.launch()
kern.decode(s, q, pages, table, lens, sk, sv, temp, again)
s.synchronize()
assert s.read_status() == [0, 0, 0, 0] and out.any() and torch.equal(out, again)
assert (narrow.float() - out.float()).abs().max() <= 2.0 ** -7 * out.float().abs().max()   # two roundings to bf16, and the weights'
g.destroy()
s.close()
print("done")
"""


def test_first_call_inside_a_capture():
    """A process whose first calls of any kind are recorded ones."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stderr[-2000:]
