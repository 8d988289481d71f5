"""The paged cache without a GPU: what its entry points refuse, and the rotation's table."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as o_paged


def _config(**kw):
    from x17ai_b200 import kernels as K
    d = dict(n_heads=8, n_kv_heads=2, head_dim=64, page_size=16, q_stride=512, kv_stride=256, o_stride=512, rotary_dim=64)
    return K.PagedConfig(**{**d, **kw})


@pytest.mark.parametrize("kw,text", [
    (dict(n_heads=0), "requires n_heads > 0"),
    (dict(n_kv_heads=0), "requires n_heads > 0"),
    (dict(n_heads=7), "multiple of n_kv_heads, got 7 and 2"),
    (dict(head_dim=48), "head_dim 32, 64 or 128, got 48"),
    (dict(page_size=8), "page_size 16, 32"),
    (dict(page_size=48), "page_size 16, 32"),
    (dict(page_size=2048), "page_size 16, 32"),
    (dict(q_stride=496), "q_stride and o_stride >="),
    (dict(o_stride=496), "q_stride and o_stride >="),
    (dict(kv_stride=240), "kv_stride >="),
    (dict(q_stride=520), "multiples of 16"),
    (dict(rotary_dim=48), "rotary_dim a multiple of 32"),
    (dict(rotary_dim=96), "rotary_dim a multiple of 32 up to head_dim"),
])
def test_configs_refused(lib, kw, text):
    from x17ai_b200 import X17Error, kernels as K
    with pytest.raises(X17Error, match=text):
        K.PagedAttnKernel(_config(**kw))


class _Stream:
    handle = 1 << 40   # never reached


class _Cuda(torch.Tensor):
    """Looks like a CUDA tensor to the checks; has no storage."""

    @staticmethod
    def __new__(cls, dtype, *shape):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError("no storage")


def _c(dtype, *shape):
    return _Cuda(dtype, *shape)


I8, I16, I32, F32, BF16 = torch.int8, torch.int16, torch.int32, torch.float32, torch.bfloat16


def _append_args(**kw):
    a = dict(q=_c(I8, 5, 512), kv=_c(I8, 5, 256), seqs=_c(I32, 5), positions=_c(I32, 5), page_table=_c(I32, 3, 4), pages=_c(I8, 9, 2, 16, 128),
             q_out=_c(I8, 5, 512), rope=_c(I16, 64, 32, 2))
    return {**a, **kw}


@pytest.mark.parametrize("kw,text", [
    (dict(kv=_c(I8, 5, 128)), "kv has 128 columns, but should have 256"),
    (dict(kv=_c(BF16, 5, 256)), "kv has dtype torch.bfloat16, but should have i8"),
    (dict(kv=_c(I8, 0, 256)), "kv has zero size"),
    (dict(seqs=_c(I32, 4)), r"seqs must have shape \[5\]"),
    (dict(positions=_c(torch.int64, 5)), "positions has dtype torch.int64"),
    (dict(page_table=_c(torch.int64, 3, 4)), "page_table has dtype torch.int64"),
    (dict(page_table=_c(I32, 3, 0)), "page_table has zero size"),
    (dict(page_table=torch.zeros((3, 4), dtype=I32)), "page_table is not on device cuda"),
    (dict(pages=_c(I8, 9, 2, 32, 128)), r"pages must have shape \[n_pages, 2, 16, 128\]"),
    (dict(pages=_c(I8, 0, 2, 16, 128)), "pages must have shape"),
    (dict(q=None), "takes q and q_out together"),
    (dict(q_out=None), "takes q and q_out together"),
    (dict(q=_c(I8, 4, 512)), "q has 4 rows, but should have 5"),
    (dict(q_out=_c(BF16, 5, 512)), "q_out has dtype torch.bfloat16"),
    (dict(kv_out=_c(I8, 5, 512)), "kv_out has 512 columns"),
    (dict(rope=None), "takes a rope table exactly where"),
    (dict(rope=_c(I16, 64, 16, 2)), r"rope must be int16 \[positions, 32, 2\]"),
    (dict(rope=_c(F32, 64, 32, 2)), "rope must be int16"),
    (dict(rope=torch.zeros((64, 32, 2), dtype=I16)), "rope must be a contiguous tensor on device cuda"),
])
def test_append_refuses(lib, kw, text):
    from x17ai_b200 import X17Error, kernels as K
    with pytest.raises(X17Error, match=text):
        K.PagedAttnKernel(_config()).append(_Stream(), **_append_args(**kw))


@pytest.mark.parametrize("kw,text", [
    (dict(page_scales=_c(F32, 9, 2, 16)), r"page_scales must have shape \[9, 2, 16, 2\]"),
    (dict(page_scales=_c(BF16, 9, 2, 16, 2)), "page_scales has dtype torch.bfloat16"),
    (dict(q_scale=None), "takes q and q_scale together"),
    (dict(q_scale=_c(F32, 5, 2)), "q_scale has 2 columns, but should have 8"),
    (dict(kv=_c(I8, 5, 256)), "kv has dtype torch.int8, but should have bf16"),
])
def test_append_scaled_refuses(lib, kw, text):
    from x17ai_b200 import X17Error, kernels as K
    args = _append_args(q=_c(BF16, 5, 512), kv=_c(BF16, 5, 256), page_scales=_c(F32, 9, 2, 16, 2), q_scale=_c(F32, 5, 8))
    with pytest.raises(X17Error, match=text):
        K.PagedAttnKernel(_config()).append_scaled(_Stream(), **{**args, **kw})


def _decode_args(**kw):
    a = dict(q=_c(I8, 6, 512), pages=_c(I8, 9, 2, 16, 128), page_table=_c(I32, 3, 4), kv_lens=_c(I32, 3), sink_k=_c(I8, 8, 64),
             sink_v=_c(I8, 8, 64), attn_temperature=_c(F32, 8), out=_c(BF16, 6, 512), l=_c(F32, 6, 8))
    return {**a, **kw}


@pytest.mark.parametrize("kw,text", [
    (dict(q=_c(I8, 7, 512)), "7 rows, which is no multiple of the 3 sequences"),
    (dict(q=_c(BF16, 6, 512)), "q has dtype torch.bfloat16"),
    (dict(kv_lens=_c(torch.int64, 3)), "kv_lens must be a contiguous int32"),
    (dict(kv_lens=_c(I32, 0)), "kv_lens must be a contiguous int32"),
    (dict(kv_lens=_c(I32, 3, 1)), "kv_lens must be a contiguous int32"),
    (dict(page_table=_c(I32, 4, 4)), "page_table has 4 rows, but should have 3"),
    (dict(sink_k=_c(I8, 2, 64)), "sink_k has 2 rows, but should have 8"),
    (dict(sink_v=_c(I8, 8, 32)), "sink_v has 32 columns, but should have 64"),
    (dict(attn_temperature=_c(F32, 2)), r"attn_temperature must have shape \[8\]"),
    (dict(out=_c(F32, 6, 512)), "out has dtype torch.float32"),
    (dict(out=_c(BF16, 3, 512)), "out has 3 rows, but should have 6"),
    (dict(l=_c(F32, 8, 6)), "l has 8 rows, but should have 6"),
    (dict(scratch=_c(I8, 1 << 20)), "scratch must be a contiguous uint8"),
    (dict(scratch=torch.zeros(1 << 20, dtype=torch.uint8)), "scratch must be a contiguous uint8"),
])
def test_decode_refuses(lib, kw, text):
    from x17ai_b200 import X17Error, kernels as K
    with pytest.raises(X17Error, match=text):
        K.PagedAttnKernel(_config()).decode(_Stream(), **_decode_args(**kw))


@pytest.mark.parametrize("kw,text", [
    (dict(out=_c(I8, 6, 512)), "out has dtype torch.int8, but should have bf16"),
    (dict(q_scale=_c(F32, 6, 2)), "q_scale has 2 columns, but should have 8"),
    (dict(page_scales=_c(F32, 8, 2, 16, 2)), r"page_scales must have shape \[9"),
])
def test_decode_scaled_refuses(lib, kw, text):
    from x17ai_b200 import X17Error, kernels as K
    args = _decode_args(q_scale=_c(F32, 6, 8), page_scales=_c(F32, 9, 2, 16, 2))
    with pytest.raises(X17Error, match=text):
        K.PagedAttnKernel(_config()).decode_scaled(_Stream(), **{**args, **kw})


def test_tensors_without_storage_raise(lib):
    """Regular arguments whose memory cannot be read: the native launch path gives them back, the Python path raises."""
    from x17ai_b200 import kernels as K
    kern = K.PagedAttnKernel(_config())
    scales, bf16 = dict(page_scales=_c(F32, 9, 2, 16, 2)), dict(q=_c(BF16, 5, 512), kv=_c(BF16, 5, 256), q_scale=_c(F32, 5, 8))
    for call in (lambda: kern.append(_Stream(), **_append_args()), lambda: kern.append_scaled(_Stream(), **_append_args(**scales, **bf16)),
                 lambda: kern.decode(_Stream(), **_decode_args()),
                 lambda: kern.decode_scaled(_Stream(), **_decode_args(**scales, q_scale=_c(F32, 6, 8)))):
        with pytest.raises(RuntimeError):
            call()


def _entry(lib, name, **kw):
    """A C entry point with plausible addresses (never read: every refusal comes before the device is entered)."""
    from x17ai_b200 import _lib
    cfg = _config(**kw.pop("cfg", {}))._c()
    p, cfg = 1 << 20, ctypes.byref(cfg)
    if name == "append":
        a = dict(stream=p, cfg=cfg, q=p, kv=p, tokens=5, seqs=p, positions=p, table=p, n_seqs=3, max_pages=4, rope=p, rope_rows=64, pages=p,
                 n_pages=9, q_out=p, kv_out=0)
        fn = lib.x17ai_b200_paged_append
    elif name == "append_scaled":
        a = dict(stream=p, cfg=cfg, q=p, kv=p, tokens=5, seqs=p, positions=p, table=p, n_seqs=3, max_pages=4, rope=p, rope_rows=64, pages=p,
                 scales=p, n_pages=9, q_out=p, q_scale=p)
        fn = lib.x17ai_b200_paged_append_scaled
    elif name == "decode":
        a = dict(stream=p, cfg=cfg, batch=3, n_tokens=2, q=p, pages=p, n_pages=9, table=p, max_pages=4, kv_lens=p, sink_k=p, sink_v=p, temp=p,
                 out=p, out_dtype=0x40, l=0, window=0, scratch=0, scratch_bytes=0)
        fn = lib.x17ai_b200_paged_decode
    else:
        a = dict(stream=p, cfg=cfg, batch=3, n_tokens=2, q=p, q_scale=p, pages=p, scales=p, n_pages=9, table=p, max_pages=4, kv_lens=p,
                 sink_k=p, sink_v=p, temp=p, out=p, l=0, window=0, scratch=0, scratch_bytes=0)
        fn = lib.x17ai_b200_paged_decode_scaled
    assert set(kw) <= set(a)
    return _lib.take_diag(fn(*{**a, **kw}.values()))


@pytest.mark.parametrize("name,kw,text", [
    ("append", dict(tokens=0), "zero size"),
    ("append", dict(n_pages=0), "must not be empty"),
    ("append", dict(max_pages=1 << 28), "out of range"),
    ("append", dict(n_pages=1 << 31), "out of range"),
    ("append", dict(kv=0), "null tensor"),
    ("append", dict(q=0), "q and its outputs come together"),
    ("append", dict(q_out=0), "q and its outputs come together"),
    ("append", dict(rope=0), "rope table"),
    ("append", dict(rope_rows=0), "rope table"),
    ("append", dict(cfg=dict(rotary_dim=0)), "rope table"),
    ("append", dict(kv=(1 << 20) + 8), "16-byte aligned"),
    ("append", dict(pages=(1 << 20) + 8), "16-byte aligned"),
    ("append", dict(cfg=dict(head_dim=48)), "head_dim 32, 64 or 128"),
    ("append", dict(stream=0), "null stream"),
    ("append_scaled", dict(scales=0), "null tensor"),
    ("append_scaled", dict(q_scale=0), "q and its outputs come together"),
    ("decode", dict(batch=0), "zero size"),
    ("decode", dict(n_tokens=0), "zero size"),
    ("decode", dict(n_tokens=65), "64 new tokens"),
    ("decode", dict(batch=65536), "at most 65535"),
    ("decode", dict(window=24), "divisible by 16, got 24"),
    ("decode", dict(out_dtype=0x50), "bf16 or FixedI8"),
    ("decode", dict(kv_lens=0), "null tensor"),
    ("decode", dict(out=(1 << 20) + 4), "16-byte aligned"),
    ("decode_scaled", dict(scales=0), "null tensor"),
    ("decode_scaled", dict(q_scale=0), "null tensor"),
])
def test_entry_points_refuse(lib, name, kw, text):
    assert text in _entry(lib, name, **kw)


def test_rope_table_is_the_angles():
    from x17ai_b200 import X17Error, kernels as K
    got = K.rope_table(70001, 64, base=500000.0, device="cpu").numpy()
    assert got.dtype == np.int16 and got.shape == (70001, 32, 2)
    assert np.array_equal(got[[0, 1, 777, 70000]], o_paged.rope_table(70001, 64, 500000.0)[[0, 1, 777, 70000]])
    assert np.array_equal(got[0, :, 0], np.full(32, 16384)) and not got[0, :, 1].any()
    for bad in ((0, 64), (10, 0), (10, 48)):
        with pytest.raises(X17Error, match="rope table requires"):
            K.rope_table(*bad, device="cpu")


def test_oracle_rotation_keeps_lengths():
    """The oracle's integer rotation against complex numbers in float64: each code within half a step of the table's angle."""
    rng = np.random.default_rng(5)
    x = rng.integers(-127, 128, (40, 3, 64), dtype=np.int8)
    x[0, 0, :2] = -128   # a code that FixedI8 never writes: clamped like any other
    cs = o_paged.rope_table(4000, 64)[rng.integers(0, 4000, 40)]
    for adjacent in (False, True):
        got = o_paged.rotate(x, cs, 64, adjacent).astype(np.float64)
        pair = lambda v: v[..., 0::2] + 1j * v[..., 1::2] if adjacent else v[..., :32] + 1j * v[..., 32:]
        z = pair(x.astype(np.float64)) * ((cs[..., 0] + 1j * cs[..., 1]) / 16384)[:, None]
        want = np.stack((z.real, z.imag)).clip(-127, 127)
        assert np.abs(np.stack((pair(got).real, pair(got).imag)) - want).max() <= 0.5
