"""The models' paths through the serving operators: BitNet's cached decoding and beams, DeepSeek-V3.2's fused norms
and beam search.  On the CPU (host forms) and, marked ``gpu``, on the device."""
import os

import pytest
import torch
import torch.multiprocessing as mp

from tilelang.models import bitnet
from tilelang.models.bitnet import BitnetConfig, BitnetForCausalLM
from tilelang.models.deepseek_v32 import ModelArgs, Transformer, generate, generate_beams
from tilelang.ops.norm import add_rms_norm_quant

on_devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def bitnet_model(device, **over):
    torch.manual_seed(0)
    cfg = BitnetConfig.tiny()
    for k, v in over.items():
        setattr(cfg, k, v)
    return BitnetForCausalLM(cfg).to(device)


def bitnet_steps(m, ids, start, page=16):
    """Logits of every position from ``start`` - 1 on, the prompt in one step and then token by token."""
    b, total = ids.shape
    pages = -(-total // page)
    heads, d = m.cfg.num_attention_heads, m.cfg.hidden_size // m.cfg.num_attention_heads
    caches = [bitnet.alloc_kv_cache(b * pages, heads, d, page, ids.device) for _ in m.layers]
    table = torch.arange(b * pages, dtype=torch.int32, device=ids.device).view(b, pages)
    lengths = torch.full((b, ), start, dtype=torch.int32, device=ids.device)
    out = [m._step(ids[:, :start], 0, caches, table, lengths)]
    for cur in range(start, total):
        lengths += 1
        out.append(m._step(ids[:, cur:cur + 1], cur, caches, table, lengths))
    return torch.stack(out, 1)


@on_devices
@pytest.mark.parametrize("over", [{}, {"num_attention_heads": 2, "hidden_size": 192}])
def test_bitnet_cached_steps_match_the_whole_sequence(device, over):
    """e4m3 keys and values are off by up to 2^-4 of themselves, 2.6 % in the root mean square; the attention's
    outputs by no more, and each of the two layers adds as much to the residual stream again: 0.15 of the logits
    leaves room for the int8 activations that flip by a step behind it."""
    m = bitnet_model(device, **over)
    ids = torch.randint(0, m.cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(1)).to(device)
    want = m(ids)[:, 20:].float()
    got = bitnet_steps(m, ids, 21).float()
    assert (got - want).norm() / want.norm() < 0.15


def test_bitnet_cached_steps_with_an_exact_cache(monkeypatch):
    """With keys and values kept as they are, positions, lengths and masks have to give the same logits but for the
    attention's rounding to fp16 (2^-11) and int8 activations that flip by one step of 127 behind it."""
    kept = {}

    def append(cache, k, v, table, lengths):
        old = kept.get(id(cache.k))
        kept[id(cache.k)] = (k.float(), v.float()) if old is None else tuple(
            torch.cat([o, n.float()], 1) for o, n in zip(old, (k, v)))

    def attend(q, cache, table, lengths):
        k, v = kept[id(cache.k)]
        assert (lengths == k.shape[1]).all()
        s = torch.einsum("bqhd,bkhd->bhqk", q.float(), k) * q.shape[-1]**-0.5
        hidden = torch.ones(q.shape[1], k.shape[1], dtype=torch.bool).triu(k.shape[1] - q.shape[1] + 1)
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        return torch.einsum("bhqk,bkhd->bqhd", p, v).to(q.dtype)

    monkeypatch.setattr(bitnet, "kv_cache_append", append)
    monkeypatch.setattr(bitnet, "kv_cache_attention", attend)
    m = bitnet_model("cpu")
    ids = torch.randint(0, m.cfg.vocab_size, (2, 30), generator=torch.Generator().manual_seed(2))
    want, got = m(ids)[:, 10:].float(), bitnet_steps(m, ids, 11).float()
    assert (got - want).norm() / want.norm() < 0.02


@on_devices
def test_bitnet_generate_cached(device):
    m = bitnet_model(device)
    ids = torch.randint(0, m.cfg.vocab_size, (2, 19), generator=torch.Generator().manual_seed(3)).to(device)
    greedy = m.generate_cached(ids, 6, page_size=16)
    assert greedy.shape == (2, 25) and torch.equal(greedy[:, :19], ids)
    # the greedy tokens are the best ones of the same cached steps
    assert torch.equal(bitnet_steps(m, greedy[:, :24], 19)[:, :6].argmax(-1), greedy[:, 19:])
    out, scores = m.generate_cached(ids, 6, beams=3, page_size=16)
    assert out.shape == (2, 3, 25) and scores.shape == (2, 3)
    assert (scores[:, :-1] >= scores[:, 1:]).all() and torch.isfinite(scores).all()
    for i in range(2):
        assert len({tuple(r) for r in out[i].tolist()}) == 3
    # the caches followed their beams: a beam's score is what its tokens get when they are decoded by themselves.
    # Only the prompt's and a beam's pages may have been scaled at other times, which changes no value but the
    # smallest ones; fp16 logits (2^-11 of up to 4) leave 2^-9 a step
    for k in range(3):
        logp = torch.log_softmax(bitnet_steps(m, out[:, k, :24], 19).float(), -1)[:, :6]
        own = logp.gather(2, out[:, k, 19:, None]).sum((1, 2))
        assert (own - scores[:, k]).abs().max() < 6 * 2.0**-6
    with pytest.raises(ValueError, match="generate_cached"):
        m.generate_cached(ids, 2, beams=33)
    with pytest.raises(ValueError, match="generate_cached"):
        m.generate_cached(ids[:, :0], 2)


@on_devices
def test_bitnet_beams_end(device):
    m = bitnet_model(device)
    ids = torch.randint(0, m.cfg.vocab_size, (1, 5), generator=torch.Generator().manual_seed(4)).to(device)
    eos = int(m.generate_cached(ids, 1)[0, -1])  # the most likely next token
    out, scores = m.generate_cached(ids, 5, beams=2, eos_id=eos, page_size=16)
    assert (out[0, 0, 5:] == eos).all()  # its score stays, and a longer one's only falls
    first = torch.log_softmax(bitnet_steps(m, ids, 5, 16)[:, 0].float(), -1)[0, eos]
    assert (scores[0, 0] - first).abs() < 2.0**-8


def deepseek(device, **over):
    return Transformer(ModelArgs.tiny(max_batch_size=6, **over), seed=0, device=device)


@on_devices
@pytest.mark.parametrize("fmt", [None, "ue8m0"])
def test_deepseek_fused_norms(device, fmt):
    """Dense layers (fp8 activations turn the tiny model's routing, fused or not): the fused norms are as far from the
    bf16 model as the separate ones may be (test_fp8_checkpoint_format_model), prefill and cached step alike."""
    toks = torch.randint(0, 512, (2, 12), generator=torch.Generator().manual_seed(5)).to(device)
    dense = dict(n_layers=2, n_dense_layers=2)
    ref = deepseek(device, **dense)(toks, 0)
    fp8 = dict(gemm_impl="fp8", norm_quant="fused", scale_fmt=fmt, **dense)
    out = deepseek(device, **fp8)(toks, 0)
    assert (out - ref).norm() / ref.norm() < 0.15
    step = deepseek(device, **fp8)
    step(toks[:, :11], 0)
    assert (step(toks[:, 11:], 11) - out).norm() / out.norm() < 0.15


@on_devices
def test_deepseek_fused_norms_in_place(device, monkeypatch):
    """Experts included: three fused norms a layer, each with the sum, the norm and the codes of its definition."""
    from test_serving_ops import check_norm
    from tilelang.models import deepseek_v32 as D
    calls = []

    def checked(x, weight, residual=None, eps=1e-6, group=128, pow2_scale=False, return_norm=False):
        r = add_rms_norm_quant(x, weight, residual, eps, group, pow2_scale, return_norm)
        check_norm(x, weight, residual, group, pow2_scale, r, eps)
        calls.append(residual is not None)
        return r

    monkeypatch.setattr(D, "add_rms_norm_quant", checked)
    toks = torch.randint(0, 512, (2, 12), generator=torch.Generator().manual_seed(5)).to(device)
    out = deepseek(device, gemm_impl="fp8", norm_quant="fused")(toks, 0)
    assert torch.isfinite(out).all() and calls == [False, False, True] * 2


def test_deepseek_norm_quant_is_checked():
    for over in (dict(norm_quant="yes"), dict(norm_quant="fused"),
                 dict(norm_quant="fused", gemm_impl="fp8", q_lora_rank=96)):
        with pytest.raises(ValueError, match="norm_quant"):
            Transformer(ModelArgs.tiny(**over), seed=0, device="cpu")


@on_devices
def test_deepseek_beams(device):
    """One beam is the greedy search; more are in order, distinct, and the cached rows their own."""
    prompts = [[1, 2, 3, 4, 5], [9, 8, 7, 6, 5]]
    greedy = generate(deepseek(device), prompts, 3)
    assert [r[0][0] for r in generate_beams(deepseek(device), prompts, 3, 1)] == greedy
    m = deepseek(device)
    got = generate_beams(m, prompts, 3, 3)
    for beams in got:
        assert len(beams) == 3 and len({tuple(t) for t, _ in beams}) == 3
        assert all(a[1] >= b[1] for a, b in zip(beams, beams[1:]))
    # the next step's logits are those of the whole sequence (to what a cached step differs from a prefill:
    # test_incremental_decode_matches_prefill)
    seqs = torch.tensor([p + t for p, beams in zip(prompts, got) for t, _ in beams], device=device)
    torch.testing.assert_close(m(seqs[:, -1:], 7), deepseek(device)(seqs, 0), rtol=3e-2, atol=3e-2)


def test_deepseek_beam_scores():
    """A score is the sum of the tokens' log probabilities; each logit may be off by 3e-2 (as above), and the
    normaliser as much."""
    one = dict(n_layers=1)
    got = generate_beams(deepseek("cpu", **one), [[1, 2, 3]], 2, 3)[0]
    seqs = torch.tensor([[1, 2, 3] + t for t, _ in got])
    total = 0.0
    for k in range(2):
        logits = deepseek("cpu", **one)(seqs[:, :3 + k], 0)
        total = total + torch.log_softmax(logits.double(), -1).gather(1, seqs[:, 3 + k:4 + k]).squeeze(1)
    assert (total - torch.tensor([s for _, s in got])).abs().max() < 2 * 2 * 3e-2


def _beams_worker(rank, world, port, prompts, out):
    import torch.distributed as dist
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.save(generate_beams(deepseek("cpu", n_layers=1), prompts, 3, 3), f"{out}.{rank}")
    finally:
        dist.destroy_process_group()


@pytest.mark.timeout(600)
def test_deepseek_beams_tensor_parallel(tmp_path):
    """Two ranks return the same beams; their scores are the log probabilities that one process gives the tokens
    (each logit and the normaliser within 3e-2 a step, as in test_deepseek_beam_scores)."""
    prompts, out = [[1, 2, 3], [9, 8, 7]], str(tmp_path / "beams")
    mp.spawn(_beams_worker, args=(2, 29500 + (os.getpid() + 977) % 2000, prompts, out), nprocs=2, join=True)
    got = [torch.load(f"{out}.{r}", weights_only=True) for r in range(2)]
    assert got[0] == got[1]
    for beams in got[0]:
        assert len(beams) == 3 and len({tuple(t) for t, _ in beams}) == 3
        assert all(a[1] >= b[1] for a, b in zip(beams, beams[1:]))
    seqs = torch.tensor([p + t for p, beams in zip(prompts, got[0]) for t, _ in beams])
    total = 0.0
    for k in range(3):
        logp = torch.log_softmax(deepseek("cpu", n_layers=1)(seqs[:, :3 + k], 0).double(), -1)
        total = total + logp.gather(1, seqs[:, 3 + k:4 + k]).squeeze(1)
    assert (total - torch.tensor([s for beams in got[0] for _, s in beams])).abs().max() < 3 * 2 * 3e-2


@pytest.mark.parametrize("call", ["beams", "cached", "cached beams"])
def test_calls_with_nothing_to_do_are_refused(call):
    """No prompts, or fewer than one new token."""
    if call == "beams":
        m = deepseek("cpu", n_layers=1)
        for prompts, new in (([], 2), ([[1, 2]], 0), ([[1, 2]], -1)):
            with pytest.raises(ValueError, match="generate_beams"):
                generate_beams(m, prompts, new, 2)
        return
    m, beams = bitnet_model("cpu"), 1 if call == "cached" else 2
    ids = torch.zeros(1, 4, dtype=torch.long)
    for prompts, new in ((ids[:0], 2), (ids, -1)) + (((ids, 0), ) if beams > 1 else ()):
        with pytest.raises(ValueError, match="generate_cached"):
            m.generate_cached(prompts, new, beams=beams)
    if beams == 1:  # as generate
        assert torch.equal(m.generate_cached(ids, 0), ids)


def test_deepseek_beams_end_and_refuse():
    m = deepseek("cpu")
    first = generate(m, [[3, 1, 4]], 1)[0][0]
    beams = generate_beams(deepseek("cpu"), [[3, 1, 4]], 6, 2, eos_id=first)[0]
    assert [first] in [t for t, _ in beams]
    for t, _ in beams:
        assert first not in t[:-1]
    for bad in (dict(prompt_tokens=[[1, 2], [3]], beams=2), dict(prompt_tokens=[[]], beams=2),
                dict(prompt_tokens=[[1]], beams=7), dict(prompt_tokens=[[1]], beams=0),
                dict(prompt_tokens=[[1]], beams=2, max_new_tokens=256)):
        with pytest.raises(ValueError, match="generate_beams"):
            generate_beams(m, **{"max_new_tokens": 2, **bad})
