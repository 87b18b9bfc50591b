"""Engines whose keys and values are cached in 8 or 4 bits, against the plain model with the same rounding (plain_quant.py)."""
import pytest
import torch

import plain_qwen3 as P
import plain_quant as Q
from gpu_util import model_folder, part_engine, plain_logits, plain_weights, random_tokens
from kipp_b200.config.base import ConfigError
from kipp_b200.engine import Engine, StepEntry
from tiny import nmse

pytestmark = pytest.mark.gpu
BITS = {"int8": 8, "int4": 4}


def engine(name, kv_quant, dtype="float32", **more):
    return Engine.from_folder(model_folder(name), dtype=dtype, kv_quant=kv_quant, **{**dict(
        page_size=16, cache_tokens=2048, max_requests=4, max_batch_tokens=512), **more})


def rounded(bits):
    """What a key or value head becomes in the cache."""
    return lambda x: Q.values(*Q.quantise(x.float(), bits), bits)


def plain(name, dtype, tokens, bits):
    cfg, w = plain_weights(name, dtype)
    with torch.no_grad():
        return P.plain_forward(cfg, w, list(tokens), kv_rounding=rounded(bits), **(P.BF16_PATH if dtype == "bfloat16" else P.F32_PATH))


def run(eng, tokens, cuts, rid="r"):
    rows, at = [], 0
    for n in cuts:
        rows.append(eng.step([StepEntry(rid, tokens[at:at + n], list(range(n)))], check=True).double().cpu())
        at += n
    return torch.cat(rows)


@pytest.mark.parametrize("kv_quant", ["int8", "int4"])
@pytest.mark.parametrize("name,page", [("B", 16), ("D", 16), ("E", 16), ("E", 6)])
def test_engine_in_32_bit(name, page, kv_quant):
    """Portions, a few tokens and single ones.  The engine's keys are off by some 1e-7, which moves the code of about one element in a
    million by a step; a step of one channel of one key is 2^-6 of that channel's mean square and a channel one of hundreds, so
    that even a moved code stays below 1e-5 of the logits."""
    tokens, cuts = random_tokens(name, 107, seed=3), (70, 3, 1, 1, 32)
    got = run(engine(name, kv_quant, page_size=page), tokens, cuts)
    want = plain(name, "float32", tokens, BITS[kv_quant])
    assert nmse(got, want) <= 1e-5
    unrounded = plain_logits(name, "float32", tokens).double()
    assert nmse(got, want) < 0.05 * nmse(unrounded, want)          # and it is this rounding that the logits show


@pytest.mark.parametrize("kv_quant", ["int8", "int4"])
@pytest.mark.parametrize("name,page", [("B", 16), ("D", 16), ("E", 16), ("E", 32), ("E", 6)])
def test_engine_in_bfloat16(name, page, kv_quant):
    """A bfloat16 step moves more codes: those whose border lies within the rounding of the projection, 2^-9 of an element against a step
    of 2^-3 (2^-7) of the group's largest, one in fifty (in three), by a step each, where the rounding to codes itself is off by a
    twelfth of a step's square: at most half as much again as the rounding does, above the bound of a bfloat16 step without it."""
    tokens, cuts = random_tokens(name, 107, seed=4), (70, 3, 1, 1, 32)
    got = run(engine(name, kv_quant, "bfloat16", page_size=page), tokens, cuts)
    want, unrounded = plain(name, "bfloat16", tokens, BITS[kv_quant]), plain_logits(name, "bfloat16", tokens).double()
    assert nmse(got, want) <= 1e-4 + 0.5 * nmse(unrounded, want)


@pytest.mark.parametrize("kv_quant", ["int8", "int4"])
@pytest.mark.parametrize("name", ["D", "E"])
def test_batches_bursts_and_graphs(name, kv_quant):
    """Requests of different lengths beside one another, a prompt beside decoded tokens, a burst that runs without the host, captured
    and replayed steps: each request's logits as when it is alone."""
    eng = engine(name, kv_quant, "bfloat16")
    texts = {r: random_tokens(name, n, seed=10 + i) for i, (r, n) in enumerate((("a", 150), ("b", 33), ("c", 7)))}
    eng.step([StepEntry(r, t[:-4], []) for r, t in texts.items()], check=True)
    rows = {r: [] for r in texts}
    for k in range(4, 0, -1):                                        # (single tokens: captured from the second step on)
        out = eng.step([StepEntry(r, [t[len(t) - k]], [0]) for r, t in texts.items()], check=True).double().cpu()
        for r, row in zip(texts, out):
            rows[r].append(row)
    late = random_tokens(name, 90, seed=20)
    both = eng.step([StepEntry("a", [5], [0]), StepEntry("d", late, [89])], check=True).double().cpu()
    alone = engine(name, kv_quant, "bfloat16", cuda_graphs=False)
    for r, t in texts.items():
        want = run(alone, t, (len(t) - 4, 1, 1, 1, 1), rid=r)[-4:]
        assert nmse(torch.stack(rows[r]), want) <= 1e-3, r
    assert nmse(both[1], run(alone, late, (90,), rid="d")[-1]) <= 1e-3
    assert eng.graph_replays > 0
    alone.finish("d")
    # the burst's tokens are those of steps that feed each row's argmax back
    for r in ("b", "c"):
        got = eng.decode_burst([r], [3], 6)
        seq, token = [], 3
        for _ in range(6):
            token = int(alone.step([StepEntry(r, [token], [0])], check=True)[0].argmax())
            seq.append(token)
        assert [int(x) for x in torch.as_tensor(got).flatten()] == seq
    eng.cache.check()


@pytest.mark.parametrize("kv_quant", ["int8", "int4"])
def test_long_portions(kv_quant):
    """Two prompts long enough for the prompt kernel over pages that are read back, beside a decoded token; then a long portion behind
    what is cached.  (The bound of test_engine_in_bfloat16.)"""
    eng = engine("E", kv_quant, "bfloat16", max_batch_tokens=1024)
    texts = {r: random_tokens("E", n, seed=30 + i) for i, (r, n) in enumerate((("a", 900), ("b", 330), ("c", 9)))}
    eng.step([StepEntry("c", texts["c"][:8], [])], check=True)
    eng.profile_start()
    out = eng.step([StepEntry("c", texts["c"][8:], [0]), StepEntry("a", texts["a"][:300], list(range(300))),
                    StepEntry("b", texts["b"], list(range(330)))], check=True).double().cpu()
    late = eng.step([StepEntry("a", texts["a"][300:], list(range(600)))], check=True).double().cpu()
    assert "attn_prefill_tc" in eng.profile_stop()
    for got, r, cut in ((out[:1], "c", slice(8, 9)), (out[1:301], "a", slice(0, 300)), (out[301:], "b", slice(0, 330)), (late, "a", slice(300, 900))):
        want, unrounded = (x[cut] for x in (plain("E", "bfloat16", texts[r], BITS[kv_quant]), plain_logits("E", "bfloat16", texts[r]).double()))
        assert nmse(got, want) <= 1e-4 + 0.5 * nmse(unrounded, want), r


def test_pages_are_reused():
    """A request on pages that others left gives what it gives on fresh ones, bit for bit, a truncated one goes on from where it was cut."""
    eng = engine("E", "int4", "bfloat16", cache_tokens=160)
    tokens = random_tokens("E", 100, seed=8)
    fresh = run(eng, tokens, (80, 1, 19), rid="x")
    eng.finish("x")
    run(eng, random_tokens("E", 150, seed=9), (150,), rid="y")
    eng.finish("y")
    again = run(eng, tokens, (80, 1, 19), rid="z")
    assert torch.equal(fresh, again)
    eng.truncate("z", 81)
    assert torch.equal(run(eng, tokens[81:], (19,), rid="z"), fresh[81:])


@pytest.mark.parametrize("kv_quant,share", [("int8", 8.5 / 16), ("int4", 4.5 / 16)])
def test_the_cache_takes_its_bits(kv_quant, share):
    eng, full = engine("E", kv_quant, "bfloat16"), engine("E", None, "bfloat16")
    info = eng.info()
    assert info["kv_bits"] == BITS[kv_quant] and full.info()["kv_bits"] == 0
    assert info["cache_bytes_per_token"] == share * full.info()["cache_bytes_per_token"]


def test_refusals():
    for name in ("A", "C"):                                          # heads of 16 and 48 channels
        with pytest.raises(ConfigError, match="multiple of 32"):
            engine(name, "int8")
    for more in (dict(kv_round_bf16=True), dict(own_length_splits=True)):
        with pytest.raises(ValueError, match="goes neither"):
            engine("E", "int4", **more)
    for bad in ("int3", 4, "q8_0"):
        with pytest.raises(ValueError, match="kv_quant"):
            engine("E", bad)


def test_a_mixer_of_another_kind_is_refused():
    from kipp_b200.parts import AttentionMixer, NoPositionEncoding, PreNormBlock, RMSNorm, SwiGLUFeedForward
    block = PreNormBlock(RMSNorm(64, 1e-5), AttentionMixer(64, 2, 1, 64, NoPositionEncoding(), value_dim=32), RMSNorm(64, 1e-5),
                         SwiGLUFeedForward(64, 16))
    with pytest.raises(ConfigError, match="plain grouped-query"):
        part_engine("bfloat16", 64, block=block, kv_quant="int8")


def test_command_line(capsys):
    from kipp_b200.cli import main
    lines = {}
    for kv in ("none", "int8", "int4"):
        assert main(["--model", model_folder("E"), "--prompt-ids", "5,17,3,9,100,7", "--decode", "8", "--kv-quant", kv]) == 0
        lines[kv] = [x for x in capsys.readouterr().out.splitlines() if x.startswith("generated")]
        assert len(lines[kv]) == 1 and len(lines[kv][0].split("\t")[1].split()) == 8


@pytest.mark.parametrize("dtype,size", [("float32", 4), ("bfloat16", 2)])
def test_the_workspace_has_room_for_an_entry_read_back(dtype, size):
    """What an engine reserves, by the message of one that is too large: beside what the plain cache's does, a whole entry of the longest
    text, where that is more than is read back at a time."""
    import re

    from kipp_b200.parts import AttentionMixer, NoPositionEncoding, PreNormBlock, RMSNorm, SwiGLUFeedForward
    reserved = {}
    for heads in (8, 640):
        for kv_quant in (None, "int8"):
            block = PreNormBlock(RMSNorm(64, 1e-5), AttentionMixer(64, heads, heads, 128, NoPositionEncoding()), RMSNorm(64, 1e-5),
                                 SwiGLUFeedForward(64, 16))
            with pytest.raises(Exception, match="of workspace") as e:
                part_engine(dtype, 64, block=block, kv_quant=kv_quant, n_pages=2 ** 27)
            reserved[heads, kv_quant] = int(re.search(r"(\d+) of workspace", str(e.value)).group(1))
    assert reserved[8, "int8"] - reserved[8, None] >= 2 ** 30
    assert reserved[640, "int8"] - reserved[640, None] >= 2 * 640 * 128 * size * 4096     # (4,096 positions)
