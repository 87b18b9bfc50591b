"""The quantised cache without a GPU: its format in plain form, and what its entry points refuse."""
from types import SimpleNamespace

import plain_quant as Q
import pytest
import torch

from kipp_b200 import kernels as K


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
def test_a_value_is_off_by_a_step_at_most(bits, D):
    """Half a step where the code is not cut off.  On the side that reaches less far the code ends at L - 1: an element as
    large as the group's largest is off by a step, and by the scale's rounding, 2^-8 of L steps, more."""
    g = torch.Generator().manual_seed(D + bits)
    x = torch.randn(50, 3, D, generator=g) * torch.exp(2 * torch.randn(50, 3, 1, generator=g))
    codes, scales = Q.quantise(x, bits)
    L = 2 ** (bits - 1)
    assert int(codes.min()) >= 0 and int(codes.max()) <= 2 * L - 1
    off = Q.groups((Q.values(codes, scales, bits) - x.double()).abs()) / scales.double().abs().unsqueeze(-1)
    assert float(off.max()) <= 1 + L * 2.0 ** -8 + 1e-6
    cut = (Q.groups(codes) == 0) | (Q.groups(codes) == 2 * L - 1)
    assert float(off[~cut].max()) <= 0.5 + 1e-6
    assert torch.equal(Q.unpack(Q.pack(codes, bits), bits), codes)


@pytest.mark.parametrize("bits", [4, 8])
def test_groups_hold_rotation_partners(bits):
    for D in (64, 128, 256):
        of = Q.groups(torch.arange(D, dtype=torch.float32))
        for row in of:
            assert sorted(((row + D // 2) % D).tolist()) == sorted(row.tolist())


@pytest.mark.parametrize("bits", [4, 8])
def test_special_values(bits):
    x = torch.zeros(6, 1, 32)
    x[1, 0, 5] = float("nan"); x[1, 0, 6] = float("inf"); x[1, 0, 7] = -3.0
    x[2, 0, 0], x[2, 0, 1] = 2.0, -2.0                       # the positive one of two alike: scale is negative
    x[3, 0, 0] = 3e38
    x[4, 0, 0] = 1e-42
    x[5] = -1.0
    codes, scales = Q.quantise(x, bits)
    v = Q.values(codes, scales, bits)
    assert torch.isfinite(v).all() and float(v[0].abs().max()) == 0
    assert v[1, 0, 7] == -3.0 and float(v[1, 0, 5:7].abs().max()) == 0
    assert float(scales[2]) < 0 and v[2, 0, 0] == 2.0
    assert v[3, 0, 0] == 2.0 ** 60
    assert (v[5] == -1.0).all()


# ------------------------------------------------------------------ refusals (nothing here reaches a kernel)
def cache(D=64, bits=4, pages=3, n_kv=2, page=8):
    return K.QuantizedPages.zeros(pages, n_kv, page, D, bits, "cpu")


@pytest.mark.parametrize("change", [dict(bits=5), dict(bits=8), dict(k_codes=torch.zeros(3, 2, 8, 16, dtype=torch.int8)),
                                    dict(k_scales=torch.zeros(3, 2, 8, 2)), dict(v_codes=torch.zeros(4, 2, 8, 32, dtype=torch.uint8)),
                                    dict(k_scales=torch.zeros(3, 2, 8, 3, dtype=torch.bfloat16)),
                                    dict(v_scales=torch.zeros(3, 2, 4, 2, dtype=torch.bfloat16)),
                                    dict(k_codes=torch.zeros(3, 2, 8, 64, dtype=torch.uint8)[..., ::2])])
def test_pages_that_do_not_fit_are_refused(change):
    c = cache()
    with pytest.raises(K.KernelError):
        K.QuantizedPages(**{**dict(k_codes=c.k_codes, k_scales=c.k_scales, v_codes=c.v_codes, v_scales=c.v_scales, bits=4), **change})


@pytest.mark.parametrize("kw", [dict(D=48), dict(D=0), dict(D=544), dict(bits=3), dict(pages=0)])
def test_sizes_that_no_cache_has(kw):
    with pytest.raises(K.KernelError):
        cache(**kw)


def write_args(T=3, nq=4, D=64, nkv=2):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)      # noqa: E731
    return dict(qkv=torch.zeros(T, (nq + 2 * nkv) * D), q_out=torch.zeros(T, nq, D), pages=cache(D=D, n_kv=nkv), q_norm_w=None,
                k_norm_w=None, eps=1e-6, inv_freq=None, rotary_dim=0, positions=i(T), entry_of_token=i(T), block_table=i(1, 2),
                tokens=T, n_q=nq, write_cache=True, status=i(4))


@pytest.mark.parametrize("change", [dict(), dict(tokens=4), dict(n_q=3), dict(q_out=torch.zeros(3, 4, 64).bfloat16()), dict(rotary_dim=3),
                                    dict(rotary_dim=66), dict(rotary_dim=64), dict(q_norm_w=torch.ones(64)),
                                    dict(q_norm_w=torch.ones(64), k_norm_w=torch.ones(32)), dict(inv_freq=torch.ones(4)),
                                    dict(positions=torch.zeros(3, dtype=torch.int64)), dict(block_table=torch.zeros(2, dtype=torch.int32)),
                                    dict(positions=torch.zeros(2, dtype=torch.int32)), dict(status=torch.zeros(3, dtype=torch.int32)),
                                    dict(cos_sin=torch.zeros(3, 8, 2), rotary_dim=64)])
def test_write_refuses(change):
    with pytest.raises(K.KernelError):                      # (with nothing changed: the tensors are not on a device)
        K.qk_norm_rope_write_quantized(**{**write_args(), **change})


def test_read_refuses():
    c, st, i = cache(), torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = torch.zeros(2, 2, 8, 64)
    for k, v, pages in ((good, good, i), (good, good.bfloat16(), i), (good[:1], good[:1], i), (good, good, i.long()),
                        (good.transpose(1, 2), good.transpose(1, 2), i)):
        with pytest.raises(K.KernelError):
            K.read_quantized_pages(k, v, c, pages, st)


@pytest.mark.parametrize("change", [dict(), dict(q=torch.zeros(2, 3, 64)), dict(q=torch.zeros(2, 4, 32)), dict(out=torch.zeros(3, 4, 64)),
                                    dict(out=torch.zeros(2, 4, 64).bfloat16()), dict(window=-1), dict(impl="other"), dict(n_q=3),
                                    dict(block_table=torch.zeros(1, 2, dtype=torch.int32)), dict(q_lens=[1, 2]),
                                    dict(q=torch.zeros(2, 4, 64).half(), out=torch.zeros(2, 4, 64).half())])
def test_attention_refuses(change):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)      # noqa: E731
    args = dict(out=torch.zeros(2, 4, 64), q=torch.zeros(2, 4, 64), pages=cache(), block_table=i(2, 2), n_q=4, scale=1.0, window=None,
                status=i(4))
    meta = SimpleNamespace(tokens=2, q_lens=change.pop("q_lens", [1, 1]), positions=i(2), entry_of_token=i(2), q_start=i(3), context_len=i(2))
    with pytest.raises(K.KernelError):
        K.attention_quantized(meta=meta, **{**args, **change})
