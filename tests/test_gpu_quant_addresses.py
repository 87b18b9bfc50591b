"""The quantised cache in tensors whose addresses are no multiples of what a kernel loads at a time."""
import pytest
import torch

from test_gpu_quant_cache import BF16, DEV, F32, attend, check, random_pages, status, step

from kipp_b200 import kernels as K

pytestmark = pytest.mark.gpu


def shifted(t):
    """A copy that begins one element behind an aligned address."""
    raw = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    raw[1:].copy_(t.flatten())
    return raw[1:].view(t.shape)


@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,nkv,page", [(64, 3, 8), (128, 2, 16), (256, 1, 4), (96, 2, 5), (32, 1, 1)])
def test_scales_two_bytes_off(D, nkv, page, bits, which):
    """Codes on 16-byte boundaries, scales at odd multiples of two bytes: what the pages give in aligned tensors."""
    layout, nq = [(70, 1), (30, 9), (0, 3)], 2 * nkv
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, D)
    odd = K.QuantizedPages(pages.k_codes, shifted(pages.k_scales) if "k" in which else pages.k_scales, pages.v_codes,
                           shifted(pages.v_scales) if "v" in which else pages.v_scales, bits)
    assert odd.k_codes.data_ptr() % 16 == 0 and (odd.k_scales.data_ptr() | odd.v_scales.data_ptr()) % 4 == 2
    order = torch.arange(n_pages, dtype=torch.int32, device=DEV)
    for dtype in (BF16, F32):
        got = [torch.empty(n_pages, nkv, page, D, dtype=dtype, device=DEV) for _ in range(2)]
        st = status()
        K.read_quantized_pages(*got, odd, order, st)
        assert torch.equal(got[0].cpu(), k.to(F32).to(dtype)) and torch.equal(got[1].cpu(), v.to(F32).to(dtype))
        q = (2 * torch.randn(meta.tokens, nq, D, generator=torch.Generator().manual_seed(1))).to(dtype).to(DEV)
        want, _ = attend(pages, meta, q, nq, D ** -0.5, impl="read")
        for impl in (None, "read"):
            out, st = attend(odd, meta, q, nq, D ** -0.5, impl=impl)
            assert torch.equal(out, want) and st.tolist() == [0] * 4
        check(out, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: True)
