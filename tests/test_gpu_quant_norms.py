"""How far attention over the quantised cache is off as a whole: a bound on the norm of a token and head's error, which a key that is
lost or a weight that is rounded too often passes where the bound of each element, with its room for cancellation, does not show it."""
import pytest
import torch

from test_gpu_quant_cache import BF16, DEV, attend, random_pages, step

pytestmark = pytest.mark.gpu

# A bfloat16 rounding of numbers whose mantissas lie anywhere is off by 2^-8 at most, and has a root mean square of 2^-8 / sqrt(3) times that of
# 1 / mantissa: 2^-8 / sqrt(3) sqrt((1 - 1/4) / (2 ln 2)) = 0.166 % of the numbers' norm.  Squares of 128 such errors, each of kurtosis 5.4
# (uniform ones, 1.8, times steps that go with Gaussian numbers, 3), have a mean that varies by sqrt(4.4 / 128) of it, its root by half of
# that: 9.3 %; five times that are allowed.  That is the result's own rounding.
# A weight p_j has one on the codes too (an eighth of one in portions, where it is float16): with S^2 = sum p_j^2 |v_j|^2 that is a root mean
# square of 0.43 * 2^-8 S, and 2^-8 S where one key has all the weight and its rounding is the worst there is; many keys' do not come
# together to more (2.4 times their root mean square, in 128 channels).  Both are independent of one another: the squares add.
ROUNDING = 2.0 ** -8 / 3 ** 0.5 * (0.75 / (2 * 0.6931472)) ** 0.5
ROOM = 1 + 5 * (4.4 / 128) ** 0.5 / 2
WEIGHTS = {"direct": 2.0 ** -8, "portion": 2.0 ** -11}


def plain(q, keys, vals, start, window, scale):
    """Q.attention's result, and S by token and head."""
    n, nq, _ = q.shape
    group = nq // keys.shape[1]
    pos, j = torch.arange(start, start + n)[:, None], torch.arange(start + n)[None]
    seen = (j <= pos) & ((j > pos - window) if window else True)
    k, v = keys.double().repeat_interleave(group, 1), vals.double().repeat_interleave(group, 1)
    p = torch.softmax((torch.einsum("nhd,jhd->hnj", q.double(), k) * scale).masked_fill(~seen, -torch.inf), -1)
    return torch.einsum("hnj,jhd->nhd", p, v), torch.einsum("hnj,jh->nh", p ** 2, (v ** 2).sum(-1)).sqrt()


@pytest.mark.parametrize("window", [None, 1100])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq,nkv,layout", [(8, 2, [(1000, 1), (2600, 1), (4099, 1)]), (16, 2, [(1500, 1)] * 6), (32, 2, [(1200, 2), (3000, 4)]),
                                           (32, 2, [(1024, 70), (2000, 130), (3000, 1)])])
def test_the_norm_of_the_error(nq, nkv, layout, bits, window):
    D, page = 128, 16
    meta, table, n_pages = step(layout, page, 7)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 7)
    q = torch.randn(meta.tokens, nq, D, generator=torch.Generator().manual_seed(7)).to(BF16).to(DEV)
    for impl in ("direct", "portion") if max(meta.q_lens) >= 64 else ("direct",):
        out, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
        assert st.tolist() == [0] * 4
        t = 0
        for e, (start, n) in enumerate(layout):
            at = table[e, :-(-(start + n) // page)].long()
            rows = lambda a: a[at].permute(0, 2, 1, 3).flatten(0, 1)[:start + n]       # noqa: E731
            want, spread = plain(q[t:t + n].cpu(), rows(k), rows(v), start, window or 0, D ** -0.5)
            far = (out[t:t + n].double().cpu() - want).norm(dim=-1)
            weights = WEIGHTS["portion" if impl == "portion" and n > 1 else "direct"]
            bound = ((ROUNDING * ROOM * want.norm(dim=-1)) ** 2 + (weights * spread) ** 2).sqrt()
            assert float((far / bound).max()) <= 1, (impl, e, float((far / bound).max()))
            t += n
