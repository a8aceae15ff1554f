"""The hand-written serving operators (tilelang._tl_ops) against their definitions in float64.

Every test runs the host form (``cpu``) and, marked ``gpu``, the gfx950 kernels.  Tolerances count roundings: a value
rounded to a type of precision ``eps`` is off by at most ``eps / 2`` of itself (bf16 2^-8, fp16 2^-11, e4m3 2^-4, and
half of e4m3's smallest step, 2^-10), float32 sums of n terms by n 2^-24 of the sum of the terms' sizes."""
import math

import pytest
import torch

from tilelang.ops.beam import beam_select, reorder_states
from tilelang.ops.kv_cache import KVCache, alloc_kv_cache, kv_cache_append, kv_cache_attention
from tilelang.ops.norm import add_rms_norm_quant

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, FP16, FP32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
on_devices = pytest.mark.parametrize("device", DEVICES)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g)


def half(t):
    return torch.finfo(t).eps / 2


def pow2_at_least(v):
    m, e = math.frexp(v)
    return math.ldexp(1.0, e - 1 if m == 0.5 else e)


# --------------------------------------------------------------------------------------------- norm


def check_norm(x, w, res, group, pow2, r, eps=1e-6):
    n, f32 = x.shape[-1], 2.0**-18  # n <= 65536 terms, summed pairwise and in parts: far below n 2^-24
    h = x.double() if res is None else x.double() + res.double()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
    if res is None:
        assert r.h is None
    else:
        assert r.h.dtype == x.dtype and ((r.h.double() - h).abs() <= (half(x.dtype) + 2.0**-24) * h.abs() + 1e-30).all()
    if r.y is not None:
        assert r.y.dtype == x.dtype
        tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
        assert ((r.y.double() - y).abs() <= (half(x.dtype) + f32) * y.abs() + tiny).all()
    parts = y.unflatten(-1, (-1, group or n))
    need = parts.abs().amax(-1).clamp_min(1e-4) / 448
    assert r.scale.dtype == FP32 and r.scale.shape == need.shape
    s = r.scale.double()
    if pow2:
        assert (torch.frexp(r.scale)[0] == 0.5).all()
        assert (s >= need * (1 - f32)).all() and (s / 2 < need * (1 + f32)).all()
    else:
        assert ((s - need).abs() <= f32 * need).all()
    assert r.q.dtype == FP8 and r.q.shape == x.shape
    got = r.q.double().unflatten(-1, (-1, group or n)) * s[..., None]
    assert ((got - parts).abs() <= (2.0**-4 + f32) * parts.abs() + 2.0**-10 * s[..., None]).all()


@on_devices
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,n,group,pow2,residual", [
    (1, 7168, 128, False, True),
    (5, 7168, 128, True, True),
    (3, 128, 128, False, False),
    (7, 16, 16, False, True),
    (2, 1536, 512, True, False),
    (4, 3200, 128, False, True),
    (9, 100, 0, False, True),
    (2, 1, 0, False, True),
    (3, 4097, 0, True, True),
    (2, 8192, 256, False, True),
    (2, 16384, 64, False, True),
    (1, 65536, 128, False, True),
    (1, 33333, 0, False, False),
    (300, 256, 32, False, True),
])
def test_norm_quant(device, dtype, rows, n, group, pow2, residual):
    g = gen(rows * n)
    x = randn(g, rows, n).to(dtype).to(device)
    res = (randn(g, rows, n) * 3).to(dtype).to(device) if residual else None
    w = (1 + randn(g, n) * 0.3).to(dtype).to(device)
    r = add_rms_norm_quant(x, w, res, group=group, pow2_scale=pow2, return_norm=True)
    check_norm(x, w, res, group, pow2, r)
    again = add_rms_norm_quant(x, w, res, group=group, pow2_scale=pow2)
    assert again.y is None and torch.equal(again.q.view(torch.uint8), r.q.view(torch.uint8))


@on_devices
def test_norm_quant_strides_and_shapes(device):
    g = gen(0)
    buf = randn(g, 6, 400).to(BF16).to(device)
    w = torch.ones(256, dtype=BF16, device=device)
    for x in (buf[:, 8:264], buf[:, 3:259], buf[::2, 8:264], buf[:, :256].t().contiguous().t(), buf[1, 8:264],
              buf[:1, :256].expand(4, 256)):
        res = (x.float() * 0.5).to(BF16)
        check_norm(x, w, res, 128, False, add_rms_norm_quant(x, w, res, return_norm=True))
    x = randn(g, 2, 3, 5, 256).to(FP16).to(device).transpose(0, 2)
    r = add_rms_norm_quant(x, w.to(FP16), None, group=64)
    assert r.q.shape == (5, 3, 2, 256) and r.scale.shape == (5, 3, 2, 4)
    check_norm(x, w.to(FP16), None, 64, False, r)
    r = add_rms_norm_quant(torch.empty(0, 256, dtype=BF16, device=device), w)
    assert r.q.shape == (0, 256) and r.scale.shape == (0, 2)


@on_devices
def test_norm_quant_zeros_and_not_finite(device):
    x = torch.zeros(4, 256, dtype=BF16, device=device)
    w = torch.ones(256, dtype=BF16, device=device)
    x[1, 7] = math.inf
    x[2, 200] = math.nan
    x[3] = 1.0
    r = add_rms_norm_quant(x, w, x, return_norm=True)
    assert (r.q[0].float() == 0).all() and (r.scale[0] == torch.tensor(1e-4) / 448).all()
    assert torch.isnan(r.q[1, 7].float()) and torch.isnan(r.y[1, 7])
    assert torch.isnan(r.q[2].float()).all()
    assert (r.q[3].float() == 448).all()


@on_devices
@pytest.mark.parametrize("group,pow2", [(128, False), (16, False), (0, False), (128, True)])
def test_norm_quant_codes_are_those_of_the_quotient(device, group, pow2):
    """Rows of +1 and -1 with eps = 0: the norm's factor is 1, y the weight with a sign, both exactly, so that scale
    and codes are what float32 divisions give (16-bit weights tie often)."""
    g = gen(21)
    n = 16384
    x = (torch.randint(0, 2, (2, n), generator=g) * 2 - 1).to(BF16)
    for dtype in (BF16, FP16, FP32):
        w = (1 + randn(g, n) * 0.4).to(BF16).to(dtype)
        r = add_rms_norm_quant(x.to(dtype).to(device), w.to(device), eps=0.0, group=group, pow2_scale=pow2)
        y = (x.float() * w.float()).unflatten(1, (-1, group or n))
        scale = y.abs().amax(-1) / 448
        if pow2:
            scale = torch.tensor([pow2_at_least(v) for v in scale.flatten().tolist()]).view(scale.shape)
        assert torch.equal(r.scale.cpu(), scale)
        want = (y / scale[..., None]).flatten(1).to(FP8)
        assert torch.equal(codes_of(r.q.view(torch.uint8)), codes_of(want.view(torch.uint8)))


@on_devices
def test_norm_quant_codes_of_zeros_and_infinite_norms(device):
    """A zero keeps its sign; a group whose largest norm is infinite has zeros beside the not-a-number."""
    x = torch.ones(1, 256, dtype=BF16, device=device)
    x[0, 1::2] = -1.0
    w = torch.ones(256, device=device).to(BF16)
    w[2:4], w[130] = 0.0, math.inf
    r = add_rms_norm_quant(x, w, eps=0.0)
    assert codes_of(r.q.view(torch.uint8))[0, 2:4].tolist() == [0, 0x80]
    rest = [i for i in range(128, 256) if i != 130]
    assert torch.isnan(r.q[0, 130].float()) and (r.q.float()[0, rest] == 0).all()
    assert (r.q.float()[0, [0, 1]].abs() == 448).all()


@on_devices
def test_norm_quant_infinite_norm_power_of_two(device):
    """The group's scale is that of the largest float32, on the host as on the device."""
    x, w = torch.ones(1, 256, dtype=BF16, device=device), torch.ones(256, dtype=BF16, device=device)
    w[130] = math.inf
    r = add_rms_norm_quant(x, w, eps=0.0, pow2_scale=True)
    assert r.scale.tolist() == [[2.0**-8, 2.0**120]]
    rest = [i for i in range(128, 256) if i != 130]
    assert torch.isnan(r.q[0, 130].float()) and (r.q.float()[0, rest] == 0).all()


@pytest.mark.gpu
def test_norm_quant_more_rows_than_a_launch_takes():
    """2^26 rows of one wave each are 2^32 threads."""
    rows, n = (1 << 26) + 5, 16
    x = torch.empty(rows, n, dtype=BF16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w = (1 + randn(gen(26), n) * 0.3).to(BF16).cuda()
    r = add_rms_norm_quant(x, w, x, group=16, return_norm=True)
    for at in (0, (1 << 21) - 2, 1 << 22, 1 << 25, rows - 4):
        part = add_rms_norm_quant(x[at:at + 4], w, x[at:at + 4], group=16, return_norm=True)
        check_norm(x[at:at + 4], w, x[at:at + 4], 16, False, part)
        for got, want in zip(r, part):
            assert torch.equal(got[at:at + 4].float(), want.float())


@on_devices
def test_norm_quant_refusals(device):
    x = torch.randn(4, 256, device=device).to(BF16)
    w = torch.ones(256, dtype=BF16, device=device)
    for err, call in (
        (TypeError, lambda: add_rms_norm_quant(x.double(), w)),
        (TypeError, lambda: add_rms_norm_quant(x, w.float())),
        (TypeError, lambda: add_rms_norm_quant(x, w, x.float())),
        (ValueError, lambda: add_rms_norm_quant(x, w[:128])),
        (ValueError, lambda: add_rms_norm_quant(x, w, x[:3])),
        (ValueError, lambda: add_rms_norm_quant(x, w, group=48)),
        (ValueError, lambda: add_rms_norm_quant(x, w, group=512)),
        (ValueError, lambda: add_rms_norm_quant(x, w, group=8)),
        (ValueError, lambda: add_rms_norm_quant(x[:, :0], w[:0], group=0)),
        (ValueError, lambda: add_rms_norm_quant(x.to("meta"), w)),
        (RuntimeError, lambda: add_rms_norm_quant(x.clone().requires_grad_(), w)),
    ):
        with pytest.raises(err, match="add_rms_norm_quant"):
            call()
    with torch.no_grad():
        add_rms_norm_quant(x.clone().requires_grad_(), w)


# --------------------------------------------------------------------------------------------- cache


def in_use(g, pages, heads, dim, page, device, junk=0x7F):
    """A cache whose every byte is ``junk`` (not-a-number codes by default) and whose scales are."""
    c = alloc_kv_cache(pages, heads, dim, page, device)
    c.k.view(torch.uint8).fill_(junk)
    c.v.view(torch.uint8).fill_(junk)
    c.k_scale.fill_(math.nan)
    c.v_scale.fill_(math.nan)
    return c


def tables(g, lens, page, width=None, spare=2):
    """Distinct pages in no order for every sequence, -1 behind them."""
    need = [-(-max(n, 0) // page) for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=g).tolist()
    t = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            t[b, i] = ids.pop()
    return t, sum(need) + spare


def ref_append(c, k, v, table, lens):
    """The definition, slot by slot, on the CPU: new pools as uint8 and scales."""
    page, dim = c.k.shape[2], c.head_dim
    out = [c.k.view(torch.uint8).cpu().clone(), c.v.view(torch.uint8).cpu().clone().transpose(2, 3).contiguous(),
           c.k_scale.cpu().clone(), c.v_scale.cpu().clone()]
    for b, end in enumerate(lens.tolist()):
        begin = end - k.shape[1]
        for nth in range(table.shape[1]):
            lo, hi = max(begin, nth * page, 0), min(end, (nth + 1) * page)
            i = int(table[b, nth])
            if hi <= lo or not 0 <= i < c.k.shape[0]:
                continue
            for which, x in enumerate((k, v)):
                new = x[b, lo - begin:hi - begin].float().cpu()  # [slot, head, dim]
                for h in range(new.shape[1]):
                    vals = new[:, h]
                    fine = vals[vals.abs() < math.inf].abs()
                    amax = max(float(fine.max()) if fine.numel() else 0.0, float(torch.tensor(1e-4)))
                    s = pow2_at_least(amax / 448)
                    slot = lo - nth * page
                    if slot:
                        old = float(out[2 + which][i, h])
                        if s > old:
                            codes = out[which][i, h, :slot].view(FP8).float() * (old / s)
                            out[which][i, h, :slot] = codes.to(FP8).view(torch.uint8)
                        s = max(s, old)
                    out[2 + which][i, h] = s
                    codes = (vals / s).clamp(-448, 448)
                    wide = torch.zeros(hi - lo, c.k.shape[3])
                    wide[:, :dim] = codes
                    out[which][i, h, slot:slot + hi - lo] = wide.to(FP8).view(torch.uint8)
    return out[0], out[1].transpose(2, 3).contiguous(), out[2], out[3]


def codes_of(x):
    """The bytes; e4m3's two codes for not-a-number (0x7f and 0xff) as one."""
    x = x.cpu()
    return torch.where(x == 0xFF, 0x7F, x.int())


def same_cache(c, ref):
    for got, want in ((c.k, ref[0]), (c.v, ref[1])):
        differ = torch.nonzero(codes_of(got.view(torch.uint8)) != codes_of(want))
        assert not len(differ), differ[:5].tolist()
    for got, want in ((c.k_scale, ref[2]), (c.v_scale, ref[3])):
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))


@on_devices
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("heads,dim,page,steps", [
    (2, 64, 16, [([20, 1, 0, 5], 20), ([21, 2, 1, 6], 1), ([30, 12, 3, 15], 10)]),
    (1, 100, 32, [([33, 64], 64), ([34, 65], 1), ([35, 66], 1)]),
    (3, 256, 64, [([100], 100), ([129], 29)]),
    (4, 128, 128, [([7, 130, -3], 130), ([8, 131, 2], 1)]),
    (1, 192, 16, [([15], 15), ([16], 1), ([17], 1)]),
    (2, 1, 16, [([5, 17], 17)]),
])
def test_append(device, dtype, heads, dim, page, steps):
    """Prompts padded on the left, then tokens one by one and in pieces that end inside pages; sizes that grow, so
    that pages are scaled again."""
    g = gen(dim * page)
    table, pages = tables(g, steps[-1][0], page)
    c = in_use(g, pages, heads, dim, page, device)
    table = table.to(device)
    for i, (lens, new) in enumerate(steps):
        lens = torch.tensor(lens, dtype=torch.int32)
        k = (randn(g, len(lens), new, heads, dim) * 4.0**i).to(dtype)
        v = (randn(g, len(lens), new, heads, dim) * 0.3 * 5.0**i).to(dtype)
        ref = ref_append(c, k, v, table.cpu(), lens)
        kv_cache_append(c, k.to(device), v.to(device), table, lens.to(device))
        same_cache(c, ref)


@on_devices
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("heads,dim,page", [(1, 256, 128), (2, 100, 1024), (1, 192, 256), (1, 64, 512), (1, 256, 1024)])
def test_append_large_pages(device, dtype, heads, dim, page):
    """Pages that no workgroup holds at once: whole ones, one that ends inside, growing scales, a token alone."""
    g = gen(dim + page)
    steps = [([page + 37, 5], page + 37), ([page + 38, 6], 1), ([2 * page, page], page - 6),
             ([2 * page + 1, page + 1], 1)]
    table, pages = tables(g, steps[-1][0], page)
    c = in_use(g, pages, heads, dim, page, device)
    table = table.to(device)
    for i, (lens, new) in enumerate(steps):
        lens = torch.tensor(lens, dtype=torch.int32)
        k = (randn(g, 2, new, heads, dim) * 4.0**i).to(dtype)
        v = (randn(g, 2, new, heads, dim) * 0.3 * 5.0**i).to(dtype)
        ref = ref_append(c, k, v, table.cpu(), lens)
        kv_cache_append(c, k.to(device), v.to(device), table, lens.to(device))
        same_cache(c, ref)
    for new, per in ((1, 4), (7, 3), (90, 1)):
        q = (randn(g, 2, new, heads * per, dim) * 2).to(FP16 if dtype == FP32 else dtype).to(device)
        check_attention(q, c, table, lens.to(device))


@on_devices
def test_append_values(device):
    """Infinities, not-a-numbers, zeros, values near the borders of a power of two, and strided inputs."""
    page, heads, dim = 16, 2, 64
    c = in_use(None, 3, heads, dim, page, device)
    table = torch.tensor([[1, 0, 2]], dtype=torch.int32, device=device)
    buf = torch.zeros(1, 6, 2, 2 * heads, dim)
    k, v = buf[:, :, 0, ::2], buf[:, :, 1, 1::2]
    k[0, 0, 0, 0], k[0, 1, 0, 3], k[0, 2, 0, 5] = math.inf, -math.inf, math.nan
    k[0, 3, 1, 1] = 448.0
    v[0, 4, 0, 0], v[0, 5, 1, 2] = 448.0 * (1 + 2.0**-23), 3e38
    moved = buf.to(device)
    for lens in (6, 12, 18):  # the second and third time into pages that hold values
        lens = torch.tensor([lens], dtype=torch.int32)
        ref = ref_append(c, k, v, table.cpu(), lens)
        kv_cache_append(c, moved[:, :, 0, ::2], moved[:, :, 1, 1::2], table, lens.to(device))
        same_cache(c, ref)
    assert float(c.k_scale[1, 1]) == 1.0 and float(c.v_scale[1, 0]) == 2.0 and float(c.v_scale[1, 1]) > 1e35


@on_devices
def test_append_leaves_the_rest(device):
    """Pages outside the pool, positions beyond the table, empty calls: nothing else is written."""
    c = in_use(None, 4, 1, 64, 16, device, junk=0x11)
    before = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8))]
    k = torch.randn(2, 40, 1, 64, device=device, dtype=BF16)
    lens = torch.tensor([40, 100], dtype=torch.int32, device=device)
    table = torch.tensor([[-1, 4, 2], [1 << 30, -5, 9]], dtype=torch.int32, device=device)
    kv_cache_append(c, k, k, table, lens)
    now = [c.k.view(torch.uint8), c.v.view(torch.uint8)]
    for old, new in zip(before, now):
        assert torch.equal(old[[0, 1, 3]], new[[0, 1, 3]])
    assert (now[0][2, :, 8:] == 0x11).all() and not (now[0][2, :, :8] == 0x11).all()
    kept = [t.clone() for t in now]
    for lens in ([0, -7], [-1, 0]):
        kv_cache_append(c, k, k, table, torch.tensor(lens, dtype=torch.int32, device=device))
    kv_cache_append(c, k[:, :0], k[:, :0], table, torch.tensor([5, 5], dtype=torch.int32, device=device))
    kv_cache_append(c, k[:0], k[:0], table[:0], torch.tensor([], dtype=torch.int32, device=device))
    assert torch.equal(kept[0], c.k.view(torch.uint8)) and torch.equal(kept[1], c.v.view(torch.uint8))


def ref_attention(q, c, table, lens, sm_scale=None):
    """float64 (out, lse, bound): bound is what roundings inside may move out by."""
    b, new, heads, d = q.shape
    page, kv = c.k.shape[2], c.k.shape[1]
    scale = d**-0.5 if sm_scale is None else sm_scale
    q, table, lens = q.double().cpu(), table.cpu(), lens.cpu()
    k8, v8 = c.k.cpu().double()[..., :d], c.v.cpu().double().transpose(2, 3)[..., :d]
    ks, vs = c.k_scale.cpu().double(), c.v_scale.cpu().double()
    out = torch.zeros(b, new, heads, d, dtype=torch.float64)
    lse = torch.full((b, new, heads), -math.inf, dtype=torch.float64)
    bound, slack = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(b):
        n = int(lens[i])
        at = torch.arange(max(min(n, table.shape[1] * page), 0))
        ids = table[i, at // page].long()
        ok = (ids >= 0) & (ids < c.k.shape[0])
        at, ids = at[ok], ids[ok]
        for h in range(heads):
            hk = h // (heads // kv)
            kk = k8[ids, hk, at % page] * ks[ids, hk, None]
            vv = v8[ids, hk, at % page] * vs[ids, hk, None]
            for t in range(new):
                m = int((at <= n - new + t).sum())
                if m == 0:
                    continue
                s = kk[:m] @ q[i, t, h] * scale
                p = torch.softmax(s, 0)
                lse[i, t, h] = torch.logsumexp(s, 0)
                out[i, t, h] = p @ vv[:m]
                # float32 scores: d products and the exponent's scaling, each off by 2^-24 of the sizes summed
                slack[i, t, h] = 2.0**-23 * (d + 8) * float((kk[:m].abs() @ q[i, t, h].abs()).max()) * abs(scale) + 1e-5
                bound[i, t, h] = p @ vv[:m].abs()
    return out, lse, bound, slack


def check_attention(q, c, table, lens, sm_scale=None):
    got, got_lse = kv_cache_attention(q, c, table, lens, sm_scale, return_lse=True)
    out, lse, bound, slack = ref_attention(q, c, table, lens, sm_scale)
    assert got.dtype == q.dtype and got.shape == q.shape and got_lse.dtype == FP32
    p_off = 2.0**-8 if q.dtype == BF16 else 2.0**-16  # the weights' rounding to bf16 (fp16: and the rest's)
    tol = (p_off + 2 * slack[..., None]) * bound + half(q.dtype) * out.abs() + torch.finfo(q.dtype).tiny
    assert ((got.double().cpu() - out).abs() <= tol).all(), float(((got.double().cpu() - out).abs() / tol).max())
    empty = lse == -math.inf
    assert torch.equal(got_lse.cpu() == -math.inf, empty) and (got.cpu()[empty] == 0).all()
    off = (got_lse.double().cpu() - lse)[~empty].abs()
    assert (off <= slack[~empty] + 1e-6 * lse[~empty].abs()).all()
    return got


def filled(g, lens, heads, dim, page, device, width=None, size=1.0):
    """A cache that holds lens tokens for each sequence, junk everywhere else."""
    table, pages = tables(g, lens, page, width)
    c = in_use(g, pages, heads, dim, page, device)
    n = max(max(lens), 1)
    lens = torch.tensor(lens, dtype=torch.int32, device=device)
    table = table.to(device)
    k = (randn(g, len(lens), n, heads, dim) * size).to(device)
    v = (randn(g, len(lens), n, heads, dim) + 0.2).to(device)
    kv_cache_append(c, k, v, table, lens)
    return c, table, lens


ATTENTION = [  # lens, new, heads, kv_heads, dim, page
    ([1], 1, 1, 1, 64, 16),
    ([70, 3, 0, 64, 65, 128], 1, 8, 2, 128, 64),
    ([300, 17], 1, 4, 4, 100, 16),
    ([257], 1, 16, 1, 64, 32),
    ([130, 129], 1, 24, 1, 128, 128),
    ([90, 33], 3, 14, 2, 80, 16),
    ([200], 1, 5, 1, 256, 64),
    ([150, 64], 2, 6, 3, 192, 32),
    ([100, 20, 5], 20, 4, 2, 128, 64),
    ([77], 77, 2, 1, 64, 16),
    ([140, 30], 40, 2, 1, 256, 64),
    ([65], 1, 2, 2, 1, 16),
    ([66, 10], 37, 7, 7, 33, 16),
]


@on_devices
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,new,heads,kv,dim,page", ATTENTION)
def test_attention(device, dtype, lens, new, heads, kv, dim, page):
    g = gen(sum(lens) + dim)
    c, table, lens = filled(g, lens, kv, dim, page, device)
    q = (randn(g, len(lens), new, heads, dim) * 2).to(dtype).to(device)
    check_attention(q, c, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,heads,kv,dim,page", [
    ([3000, 17, 1999], 1, 32, 8, 128, 64),
    ([5000], 1, 8, 8, 64, 16),
    ([2049], 4, 16, 1, 128, 32),
    ([1500, 700], 200, 8, 2, 128, 64),
    ([900], 300, 4, 4, 64, 128),
    ([700, 600], 150, 2, 1, 192, 64),
])
def test_attention_long(lens, new, heads, kv, dim, page):
    """Long axes that several workgroups share, and chunks of prompts."""
    g = gen(sum(lens))
    c, table, lens = filled(g, lens, kv, dim, page, "cuda")
    q = (randn(g, len(lens), new, heads, dim) * 2).to(BF16).to("cuda")
    check_attention(q, c, table, lens)
    check_attention(q.to(FP16), c, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,new,heads,kv,dim,page", [
    ([2100, 1900] * 8, 40, 32, 8, 128, 64),  # 128 rows to a workgroup, the key axis in one part
    ([4096, 509], 509, 32, 8, 128, 64),
    ([3000], 700, 16, 2, 80, 16),
    ([9000, 130], 130, 8, 2, 128, 32),
    ([900], 300, 32, 8, 64, 16),
    ([2000, 50], 50, 12, 2, 200, 128),
])
def test_attention_chunks(dtype, lens, new, heads, kv, dim, page):
    """Prompts' chunks at full size, against float64 on the device."""
    g = gen(sum(lens))
    c, table, lens = filled(g, lens, kv, dim, page, "cuda")
    q = (randn(g, len(lens), new, heads, dim) * 1.5).to(dtype).cuda()
    got, got_lse = kv_cache_attention(q, c, table, lens, return_lse=True)
    per = heads // kv
    for b, n in enumerate(lens.tolist()):
        ids = table[b, :-(-n // page)].long()

        def values(pool, scale):
            x = pool.view(torch.uint8)[ids].view(FP8).double() * scale[ids][..., None, None].double()
            return x.transpose(0, 1)  # [head, page, ..]

        k = values(c.k, c.k_scale).flatten(1, 2)[:, :n, :dim]
        v = values(c.v, c.v_scale).transpose(2, 3).flatten(1, 2)[:, :n, :dim].contiguous()
        x = q[b].double().view(new, kv, per, dim).permute(1, 0, 2, 3).flatten(1, 2)
        s = (x @ k.transpose(1, 2).contiguous()) * dim**-0.5
        size = (x.abs() @ k.abs().transpose(1, 2).contiguous()).amax(-1) * dim**-0.5
        row = torch.arange(new, device="cuda").repeat_interleave(per)
        hidden = torch.arange(n, device="cuda") > (n - new + row)[:, None]
        s = s.masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1)
        out, bound, lse = p @ v, p @ v.abs(), torch.logsumexp(s, -1)
        slack = 2.0**-23 * (dim + 8) * size + 1e-5
        tol = ((2.0**-8 if dtype == BF16 else 2.0**-16) + 2 * slack[..., None]) * bound
        tol = tol + half(dtype) * out.abs() + torch.finfo(dtype).tiny

        def rows(t):
            return t.double().unflatten(1, (kv, per)).transpose(0, 1).flatten(1, 2)

        assert ((rows(got[b]) - out).abs() <= tol).all()
        assert ((rows(got_lse[b]) - lse).abs() <= slack + 1e-6 * lse.abs()).all()


@pytest.mark.gpu
def test_cache_beyond_32_bits():
    """Pools of over 4 GB: the pages with the highest ids."""
    page, heads, dim = 64, 8, 128
    c = alloc_kv_cache(70000, heads, dim, page)
    assert c.k.numel() > 1 << 32
    table = torch.tensor([[69999, 2, 65600], [68000, 69998, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([190, 130], dtype=torch.int32, device="cuda")
    g = gen(9)
    k, v = randn(g, 2, 190, heads, dim).cuda(), randn(g, 2, 190, heads, dim).cuda()
    kv_cache_append(c, k, v, table, lens)
    few = torch.tensor([0, 2, 65600, 68000, 69998, 69999], device="cuda")
    small = KVCache(*(t.view(torch.uint8)[few].view(FP8) if t.dtype is FP8 else t[few] for t in c[:4]), dim)
    near = torch.tensor([[5, 1, 2], [3, 4, 0]], dtype=torch.int32, device="cuda")
    for new, per in ((1, 2), (40, 2)):
        q = randn(g, 2, new, heads * per, dim).to(BF16).cuda()
        assert torch.equal(kv_cache_attention(q, c, table, lens), check_attention(q, small, near, lens))


@on_devices
def test_attention_strides_scale_and_wide_table(device):
    g = gen(5)
    c, table, lens = filled(g, [50, 100], 2, 64, 16, device, width=40)
    qkv = randn(g, 2, 2, 12, 64).to(BF16).to(device)
    check_attention(qkv[:, :, 2:10:2], c, table, lens, 0.3)
    check_attention(qkv.transpose(1, 2)[:, :2].transpose(1, 2).expand(2, 2, 2, 64), c, table[:, :9], lens, -0.2)
    odd = randn(g, 2, 1, 4, 65).to(FP16).to(device)[..., 1:]
    check_attention(odd, c, table, lens)
    assert kv_cache_attention(qkv[:, :0, :2], c, table, lens).shape == (2, 0, 2, 64)
    assert kv_cache_attention(qkv[:0, :, :2], c, table[:0], lens[:0]).shape == (0, 2, 2, 64)
    none = kv_cache_attention(qkv[:, :, :2], c, table[:, :0], lens)
    assert (none == 0).all()


@on_devices
def test_attention_absent_pages(device):
    """Ids outside the pool are not followed; a hole in the table hides its tokens."""
    g = gen(6)
    c, table, lens = filled(g, [100, 60], 1, 64, 16, device)
    q = randn(g, 2, 2, 4, 64).to(BF16).to(device)
    for hole, value in ((0, -1), (3, 1 << 30), (6, c.k.shape[0])):
        t = table.clone()
        t[0, hole] = value
        check_attention(q, c, t, lens)
    t = table.clone()
    t[1] = -1
    assert (check_attention(q, c, t, lens)[1] == 0).all()
    check_attention(q, c, table, torch.tensor([-5, 1], dtype=torch.int32, device=device))
    c, table, lens = filled(g, [96, 96], 1, 64, 16, device)
    check_attention(q, c, table, torch.tensor([(1 << 31) - 1, 97], dtype=torch.int32, device=device))


def widened(table, page, tokens=1 << 18):
    """The same table with room for many more tokens: a long axis is prepared for (128 rows to a workgroup, many
    parts), whatever is there."""
    return torch.nn.functional.pad(table, (0, tokens // page - table.shape[1]), value=-1)


@on_devices
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,heads,kv,dim", [(40, 4, 1, 64), (33, 2, 2, 128), (20, 16, 2, 100), (30, 1, 1, 256)])
def test_attention_absent_pages_in_chunks(device, page, new, heads, kv, dim):
    """Holes of the table where every row would see the page, and where only some would."""
    g = gen(new + dim)
    c, table, lens = filled(g, [300, 170], kv, dim, page, device)
    q = randn(g, 2, new, heads, dim).to(BF16).to(device)
    t = table.clone()
    t[0, 1], t[0, 300 // page], t[1, 170 // page] = -1, 1 << 30, -7
    for table in (t, widened(t, page)):
        check_attention(q, c, table, lens)
        check_attention(q.to(FP16), c, table, lens)


@on_devices
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,heads,dim", [(7, 2, 64), (40, 1, 128), (30, 4, 100)])
def test_attention_not_finite_in_hidden_places(device, page, new, heads, dim):
    """A not-a-number in a later token's value or key reaches only the queries that see it."""
    g = gen(7)
    n = 90
    table, pages = tables(g, [n], page)
    table, lens = table.to(device), torch.tensor([n], dtype=torch.int32, device=device)
    k, v = randn(g, 1, n, 1, dim), randn(g, 1, n, 1, dim)
    clean = in_use(g, pages, 1, dim, page, device)
    kv_cache_append(clean, k.to(device), v.to(device), table, lens)
    k[0, n - 2, 0, 3] = math.nan
    v[0, n - 3, 0, 5] = math.nan
    v[0, n - 1, 0, 9] = math.nan
    c = in_use(g, pages, 1, dim, page, device)
    kv_cache_append(c, k.to(device), v.to(device), table, lens)
    q = randn(g, 1, new, heads, dim).to(BF16).to(device)
    if heads > 2:
        table = widened(table, page)
    want, got = kv_cache_attention(q, clean, table, lens), kv_cache_attention(q, c, table, lens)
    assert torch.equal(got[:, :new - 3], want[:, :new - 3])
    assert torch.isnan(got[:, new - 3, :, 5]).all()  # this query sees one such value
    rest = [d for d in range(dim) if d != 5]
    assert torch.equal(got[:, new - 3][..., rest], want[:, new - 3][..., rest])
    assert torch.isnan(got[:, new - 2:]).all()  # and these a key that is none


@on_devices
def test_attention_extreme_scales(device):
    """Pages whose scales differ by hundreds of binades, codes at both ends of e4m3, scores far apart."""
    g = gen(8)
    c, table, lens = filled(g, [64, 48], 2, 64, 16, device)
    c.v_scale.copy_(2.0**torch.randint(-60, 40, c.v_scale.shape, generator=g).float())
    c.k_scale.copy_(2.0**torch.randint(-20, 2, c.k_scale.shape, generator=g).float())
    q = (randn(g, 2, 1, 4, 64)).to(BF16).to(device)
    check_attention(q, c, table, lens)


@on_devices
@pytest.mark.parametrize("new,heads,kv", [(1, 4, 2), (24, 4, 2), (70, 4, 1)])
def test_attention_largest_values(device, new, heads, kv):
    """Values close to the type's largest: their weighted means are finite, the sums of many are not."""
    g = gen(22)
    table, pages = tables(g, [300, 90], 16)
    table, lens = table.to(device), torch.tensor([300, 90], dtype=torch.int32, device=device)
    c = in_use(g, pages, kv, 128, 16, device)
    k, v = randn(g, 2, 300, kv, 128).to(BF16), (1 + torch.rand(2, 300, kv, 128, generator=g)).mul(2.0**126).to(BF16)
    kv_cache_append(c, k.to(device), v.to(device), table, lens)
    q = randn(g, 2, new, heads, 128).to(BF16).to(device)
    for t in (table, widened(table, 16)):
        assert torch.isfinite(check_attention(q, c, t, lens)).all()


@on_devices
def test_attention_scale_must_be_finite(device):
    """A not-a-number scale gave the mean of the values on the device and not-a-numbers on the host."""
    c, table, lens = filled(gen(24), [20], 1, 64, 16, device)
    q = randn(gen(25), 1, 1, 2, 64).to(BF16).to(device)
    for bad in (math.nan, math.inf, -math.inf, 1e39):
        with pytest.raises(ValueError, match="kv_cache_attention: sm_scale"):
            kv_cache_attention(q, c, table, lens, bad)
    check_attention(q, c, table, lens, 0.0)
    check_attention(q, c, table, lens, 1e-30)


@on_devices
def test_cache_refusals(device):
    c = alloc_kv_cache(4, 2, 64, 16, device)
    table = torch.zeros(1, 4, dtype=torch.int32, device=device)
    lens = torch.tensor([3], dtype=torch.int32, device=device)
    q = torch.randn(1, 1, 4, 64, device=device).to(BF16)
    k = q[:, :, :2]

    def attend(q=q, c=c, table=table, lens=lens):
        return kv_cache_attention(q, c, table, lens)

    for err, call in (
        (TypeError, lambda: attend(q=q.float())),
        (TypeError, lambda: attend(lens=lens.long())),
        (TypeError, lambda: attend(table=table.long())),
        (TypeError, lambda: attend(c=c._replace(k=c.k.view(torch.uint8)))),
        (TypeError, lambda: attend(c=c._replace(k_scale=c.k_scale.double()))),
        (ValueError, lambda: attend(q=q[0])),
        (ValueError, lambda: attend(q=q[:, :, :3])),
        (ValueError, lambda: attend(q=q[..., :63])),
        (ValueError, lambda: attend(table=table.expand(2, 4))),
        (ValueError, lambda: attend(lens=lens.expand(2))),
        (ValueError, lambda: attend(c=c._replace(v=c.k))),
        (ValueError, lambda: attend(c=c._replace(head_dim=65))),
        (ValueError, lambda: attend(c=c._replace(k_scale=c.k_scale[:3]))),
        (ValueError, lambda: attend(c=c._replace(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)))),
        (ValueError, lambda: attend(table=torch.zeros(1, 8, dtype=torch.int32, device=device)[:, ::2])),
        (ValueError, lambda: attend(lens=lens.to("meta"))),
        (RuntimeError, lambda: attend(q=q.clone().requires_grad_())),
    ):
        with pytest.raises(err, match="kv_cache_attention"):
            call()
    for err, call in (
        (TypeError, lambda: kv_cache_append(c, k, k.float(), table, lens)),
        (ValueError, lambda: kv_cache_append(c, k, k[:, :, :1], table, lens)),
        (ValueError, lambda: kv_cache_append(c, q, q, table, lens)),
        (ValueError, lambda: kv_cache_append(c, k[..., :32], k[..., :32], table, lens)),
    ):
        with pytest.raises(err, match="kv_cache_append"):
            call()
    square = alloc_kv_cache(4, 2, 64, 64, device)
    for same in (dict(v=square.k), dict(v_scale=square.k_scale)):
        with pytest.raises(ValueError, match="share memory"):
            kv_cache_append(square._replace(**same), k, k, table, lens)
    for bad in ((4, 2, 257, 16), (4, 2, 0, 16), (4, 2, 64, 24), (4, 2, 64, 8)):
        with pytest.raises(ValueError, match="alloc_kv_cache"):
            alloc_kv_cache(*bad, device=device)


@on_devices
def test_cache_memory_that_is_shared(device):
    """What a call writes may meet nothing else that it reads or writes, not by one byte."""
    square = alloc_kv_cache(4, 2, 64, 64, device)
    table = torch.zeros(1, 4, dtype=torch.int32, device=device)
    lens = torch.tensor([3], dtype=torch.int32, device=device)
    k = torch.randn(1, 1, 2, 64, device=device).to(BF16)
    n, m = square.k.numel(), square.k_scale.numel()
    buf = torch.zeros(2 * n + 4 * 64, dtype=torch.uint8, device=device)
    floats = torch.ones(2 * m, device=device)

    def pool(at):
        return buf[at:at + n].view(FP8).view(4, 2, 64, 64)

    def scale(at):
        return floats[at:at + m].view(4, 2)

    apart = KVCache(pool(0), pool(n), scale(0), scale(m), 64)
    kv_cache_append(apart, k, k, table, lens)
    tail = buf[n - 256:n].view(BF16).view(1, 1, 2, 64)  # new tokens in K's last bytes
    ints = apart.k_scale.view(torch.int32)
    for bad, args in ((dict(v=pool(n - 64)), ()), (dict(v=pool(0)), ()), (dict(v_scale=scale(m - 1)), ()),
                      (dict(k_scale=buf[n - 64:n - 64 + 4 * m].view(FP32).view(4, 2)), ()),
                      (dict(), (tail, k, table, lens)), (dict(), (k, tail, table, lens)),
                      (dict(), (k, k, ints[:1], lens)), (dict(), (k, k, table, ints[0, :1]))):
        with pytest.raises(ValueError, match="kv_cache_append.*share memory"):
            kv_cache_append(apart._replace(**bad), *(args or (k, k, table, lens)))
    with pytest.raises(ValueError, match="kv_cache_attention.*share memory"):
        kv_cache_attention(k, apart._replace(v=pool(n - 64)), table, lens)


# --------------------------------------------------------------------------------------------- beams


def ref_select(logits, scores, take, finished=None, eos=-1):
    b, k = scores.shape
    x = logits.reshape(b, k, -1).double().cpu()
    s = scores.double().cpu()
    v = s[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    dead = torch.isnan(x).any(-1) | (x == math.inf).any(-1) | ~torch.isfinite(s)
    v = torch.where(torch.isnan(v) | dead[..., None], -math.inf, v)
    if finished is not None:
        done = finished.cpu() & torch.isfinite(s)
        v[done] = -math.inf
        v[..., eos] = torch.where(done, s, v[..., eos])
    v, at = torch.sort(v.flatten(1), dim=-1, descending=True, stable=True)
    return v[:, :take], at[:, :take] // x.shape[-1], at[:, :take] % x.shape[-1]


def check_select(logits, scores, take=None, finished=None, eos=-1):
    got = beam_select(logits, scores, take, finished, eos)
    want = ref_select(logits, scores, take or scores.shape[1], finished, eos)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    v = want[0]
    off = (got[0].double().cpu() - v).abs()
    assert torch.equal(got[0].cpu() == -math.inf, v == -math.inf)
    # the sum of float32 exponentials (each off by a few 2^-24, summed in parts) and the result's own rounding
    assert (off[v > -math.inf] <= 2.0**-20 + 2.0**-24 * v[v > -math.inf].abs()).all()


@on_devices
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("b,k,vocab,take", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 20), (1, 4, 512, 8), (3, 2, 4097, 4), (2, 8, 5000, 16), (1, 5, 32002, 10),
    (1, 16, 1000, 64), (2, 64, 33, 64),
])
def test_beam_select(device, dtype, b, k, vocab, take):
    """16-bit logits tie all the time: the lowest index wins."""
    g = gen(vocab + take)
    logits = (randn(g, b, k, vocab) * 3).to(dtype).to(device)
    scores = (-randn(g, b, k).abs() * 4).to(device)
    check_select(logits, scores, take)
    check_select(logits.view(b * k, vocab), scores, take)
    finished = (torch.rand(b, k, generator=g) < 0.4).to(device)
    check_select(logits, scores, take, finished, vocab // 2)


@pytest.mark.gpu
@pytest.mark.parametrize("b,k,vocab,take,dtype", [
    (4, 8, 129280, 16, FP32), (1, 4, 129280, 8, FP32), (2, 16, 150001, 32, BF16), (1, 2, 32002, 64, FP16),
    (40, 4, 32002, 8, FP16), (1, 64, 262144, 64, BF16), (1, 3, 262145, 6, FP32), (1, 2, 1 << 20, 4, BF16),
])
def test_beam_select_large(b, k, vocab, take, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.empty(b, k, vocab, dtype=dtype, device="cuda").normal_(0, 3, generator=g)
    scores = -torch.empty(b, k, device="cuda").normal_(0, 3, generator=g).abs()
    check_select(logits, scores, take)


@on_devices
def test_beam_select_ties_and_not_finite(device):
    g = gen(3)
    scores = torch.tensor([[0.0, -1.0, -2.0, -math.inf]], device=device)
    same = torch.zeros(1, 4, 9000, device=device)
    check_select(same, scores, 60)  # every token of a beam ties
    check_select(same, torch.zeros(1, 4, device=device), 60)  # and every beam
    check_select(torch.where(torch.arange(9000, device=device) % 2 == 0, 0.0, -0.0).expand(1, 4, 9000).contiguous(),
                 scores, 16)  # -0 ties with 0
    x = randn(g, 1, 4, 9000).to(device)
    x[0, 0, 17], x[0, 1, 8999] = math.nan, math.inf
    x[0, 2, 3:] = -math.inf
    check_select(x, scores, 12)  # two beams that come last, one with three tokens
    x[0, 2] = -math.inf
    check_select(x, scores, 12)
    check_select(x, torch.tensor([[math.inf, -math.inf, math.nan, 0.0]], device=device), 12)
    done = torch.tensor([[True, True, False, True]], device=device)
    check_select(x, scores, 40, done, 0)
    check_select(x, scores, 40, done, 8999)
    low = torch.full((1, 4, 9000), torch.finfo(FP32).min, device=device)
    check_select(low, scores, 8)
    check_select(torch.arange(9000.0, device=device).expand(1, 4, 9000), scores, 64)  # sorted, not contiguous


@on_devices
def test_beam_select_many_ties(device):
    """More candidates that tie than are kept anywhere: many beams, their rows constant or of two values."""
    zero = torch.zeros(1, 64, device=device)
    same = torch.zeros(1, 64, 5000, device=device)
    check_select(same, zero, 64)
    same[:, :, ::3] = 1.0
    check_select(same, zero, 64)
    same[:, ::2] = -math.inf
    check_select(same, zero, 64)


@on_devices
def test_beam_select_strides(device):
    g = gen(4)
    wide = randn(g, 6, 1003).to(BF16).to(device)
    scores = -randn(g, 2, 3).abs().to(device)
    check_select(wide[:, 1:1001], scores, 6)
    check_select(wide[:, :1000], scores.t().contiguous().t(), 6)
    assert beam_select(wide[:0], scores[:0], 2)[0].shape == (0, 2)


@on_devices
def test_beam_select_refusals(device):
    x, s = torch.randn(2, 3, 50, device=device), torch.zeros(2, 3, device=device)
    fin = torch.zeros(2, 3, dtype=torch.bool, device=device)
    for err, call in (
        (TypeError, lambda: beam_select(x.double(), s)),
        (TypeError, lambda: beam_select(x, s.to(BF16))),
        (TypeError, lambda: beam_select(x, s, finished=fin.int(), eos_id=1)),
        (ValueError, lambda: beam_select(x[:1], s)),
        (ValueError, lambda: beam_select(x, s, 0)),
        (ValueError, lambda: beam_select(x, s, 65)),
        (ValueError, lambda: beam_select(x[..., :2], s, 7)),
        (ValueError, lambda: beam_select(x, s, finished=fin)),
        (ValueError, lambda: beam_select(x, s, finished=fin, eos_id=50)),
        (ValueError, lambda: beam_select(x, s, finished=fin[:1], eos_id=1)),
        (ValueError, lambda: beam_select(x, s.to("meta"))),
        (RuntimeError, lambda: beam_select(x.clone().requires_grad_(), s)),
    ):
        with pytest.raises(err, match="beam_select"):
            call()


def ref_reorder(states, parents, length):
    b, k = parents.shape
    p = parents.cpu()
    rows = torch.where((p >= 0) & (p < k), p, torch.arange(k)) + k * torch.arange(b)[:, None]
    out = []
    for s in states:
        t = s.cpu().clone()
        t = t.view(torch.uint8) if t.dtype is FP8 else t
        if length is None:
            t = t[rows.flatten()]
        else:
            t[:, :length] = t[rows.flatten()][:, :length]
        out.append(t)
    return out


@on_devices
@pytest.mark.parametrize("b,k", [(1, 1), (2, 2), (1, 3), (3, 4), (2, 7), (1, 8), (2, 16), (1, 32)])
@pytest.mark.parametrize("length", [None, 0, 1, 13])
def test_reorder(device, b, k, length):
    g = gen(b * k)
    n = b * k
    for parents in (torch.randint(0, k, (b, k), generator=g), torch.zeros(b, k, dtype=torch.long),
                    torch.arange(k).flip(0).expand(b, k).contiguous(), torch.arange(k).expand(b, k).contiguous(),
                    torch.randint(-2, k + 2, (b, k), generator=g)):
        states = [randn(g, n, 20, 33), randn(g, n, 20, 64).to(BF16), randn(g, n, 20, 7).to(FP8), randn(g, n, 20),
                  torch.randint(0, 99, (n, 20), generator=g), randn(g, n, 40, 3)[:, :20],
                  torch.randint(0, 2, (n, 21, 5), generator=g, dtype=torch.uint8)[:, 1:]]
        here = [torch.empty_strided(s.size(), s.stride(), dtype=s.dtype, device=device).copy_(s) for s in states]
        want = ref_reorder(here, parents, length)
        reorder_states(here, parents.to(device), length)
        for got, ref in zip(here, want):
            got = got.view(torch.uint8) if got.dtype is FP8 else got
            assert torch.equal(got.cpu(), ref)


@on_devices
def test_reorder_many_states_and_columns(device):
    """More states than one launch takes, and two that are columns of one buffer."""
    g = gen(1)
    parents = torch.tensor([[2, 2, 0]])
    states = [randn(g, 3, 5 + i % 3).to(device) for i in range(200)]
    both = randn(g, 3, 24).to(device)
    states += [both[:, :10], both[:, 10:24]]
    want = ref_reorder(states, parents, None)
    reorder_states(states, parents.to(device))
    for got, ref in zip(states, want):
        assert torch.equal(got.cpu(), ref)


@pytest.mark.gpu
def test_reorder_more_than_a_launch_takes():
    """Two states of 32 GB and a little for each of two beams: 2^26 workgroups of one wave, 2^32 threads."""
    n = (1 << 35) + 4096
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 4 * n + (8 << 30):
        pytest.skip("needs 146 GB")
    states = [torch.empty(2, n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    at = (0, 1 << 32, n - 64)
    for i, s in enumerate(states):
        for j, p in enumerate(at):
            s[0, p:p + 64], s[1, p:p + 64] = 1, 10 * (i + 1) + j
    reorder_states(states, torch.tensor([[1, 1]], device="cuda"))
    for i, s in enumerate(states):
        for j, p in enumerate(at):
            assert (s[:, p:p + 64] == 10 * (i + 1) + j).all()
    del states, s
    torch.cuda.empty_cache()


def test_reorder_rows_that_no_launch_takes(tmp_path):
    """Refused before anything moves: rows of 2^36 bytes, in a sparse file that nobody reads or writes."""
    n = 1 << 36
    try:
        with open(tmp_path / "state", "wb") as f:
            f.truncate(2 * n)
        huge = torch.from_file(str(tmp_path / "state"), shared=True, size=2 * n, dtype=torch.uint8).view(2, n)
    except (OSError, RuntimeError) as e:
        pytest.skip(f"no sparse file of 128 GB here: {e}")
    small = torch.arange(2.0).view(2, 1)
    with pytest.raises(ValueError, match="reorder_states: 68719476736 bytes of a state's row"):
        reorder_states([small, huge], torch.tensor([[1, 1]]))
    assert small.tolist() == [[0.0], [1.0]]
    reorder_states([small, huge], torch.tensor([[1, 1]]), 1)  # what moves of a row counts


@on_devices
def test_reorder_refusals(device):
    x, p = torch.randn(6, 10, 4, device=device), torch.zeros(2, 3, dtype=torch.long, device=device)
    for err, call in (
        (TypeError, lambda: reorder_states([x], p.int())),
        (ValueError, lambda: reorder_states([x], p.flatten())),
        (ValueError, lambda: reorder_states([x[:5]], p)),
        (ValueError, lambda: reorder_states([x], p, 11)),
        (ValueError, lambda: reorder_states([x], p, -1)),
        (ValueError, lambda: reorder_states([x[:, 0, 0]], p, 1)),
        (ValueError, lambda: reorder_states([x.transpose(1, 2)], p)),
        (ValueError, lambda: reorder_states([x[:1].expand(6, 10, 4)], p)),
        (ValueError, lambda: reorder_states([x, x], p)),
        (ValueError, lambda: reorder_states([x[:, :6], x[:, 5:]], p)),
        (ValueError, lambda: reorder_states([x.to("meta")], p)),
        (ValueError, lambda: reorder_states([torch.randn(66, 2, device=device)],
                                            torch.zeros(2, 33, dtype=torch.long, device=device))),
        (RuntimeError, lambda: reorder_states([x.clone().requires_grad_()], p)),
    ):
        with pytest.raises(err, match="reorder_states"):
            call()
    with pytest.raises(ValueError, match="parents and a state share memory"):
        q = torch.zeros(6, dtype=torch.long, device=device)
        reorder_states([q], q.view(2, 3))
    reorder_states([], p)


@on_devices
def test_tensors_without_memory_are_refused(device):
    """Fake, functional and batched tensors, lazy zeros, sparse ones, alone or beside real ones."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w = torch.randn(4, 128, device=device).to(BF16), torch.ones(128, device=device).to(BF16)
    cache = alloc_kv_cache(2, 1, 64, 16, device)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device=device), torch.ones(1, dtype=torch.int32, device=device)
    kv, scores = x[:1, None, None, :64], torch.zeros(2, 2, device=device)
    parents = torch.zeros(2, 2, dtype=torch.long, device=device)
    calls = [("add_rms_norm_quant", lambda f: add_rms_norm_quant(f(x), w)),
             ("add_rms_norm_quant", lambda f: add_rms_norm_quant(x, f(w))),
             ("add_rms_norm_quant", lambda f: add_rms_norm_quant(x, w, f(x))),
             ("kv_cache_append", lambda f: kv_cache_append(cache, f(kv), f(kv), table, lens)),
             ("kv_cache_attention", lambda f: kv_cache_attention(f(kv), cache, table, lens)),
             ("kv_cache_attention", lambda f: kv_cache_attention(kv, cache, table, f(lens))),
             ("beam_select", lambda f: beam_select(f(x), scores)),
             ("beam_select", lambda f: beam_select(x, f(scores))),
             ("reorder_states", lambda f: reorder_states([x, f(x + 1)], parents)),
             ("reorder_states", lambda f: reorder_states([x], f(parents)))]

    def refused(call, name, f):
        with pytest.raises((ValueError, RuntimeError), match=name):
            call(f)

    for name, call in calls:
        mode = FakeTensorMode()
        refused(call, name, mode.from_tensor)
        with pytest.raises(Exception), mode:  # whatever meets the real tensors first
            call(mode.from_tensor)
        refused(call, name, lambda t: torch._efficientzerotensor(t.shape, dtype=t.dtype, device=device))
        refused(call, name, lambda t: t.to_sparse())
        torch.func.functionalize(lambda t: refused(call, name, torch._to_functional_tensor))(x)
    for wrap in (torch.func.functionalize, torch.vmap):
        with pytest.raises((ValueError, RuntimeError), match="null data pointer"):
            wrap(lambda t: add_rms_norm_quant(t, w).q)(x[None] if wrap is torch.vmap else x)
    with FakeTensorMode():  # real tensors are what they are inside such a mode
        reorder_states([x], parents)


@on_devices
def test_writes_are_seen_by_autograd(device):
    """A backward that saved what a call overwrites raises, instead of a gradient from the new values."""
    g = gen(23)
    c = alloc_kv_cache(2, 1, 64, 16, device)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device=device), torch.ones(1, dtype=torch.int32, device=device)
    state, k = randn(g, 4, 5).to(device), randn(g, 1, 1, 1, 64).to(device)
    parents = torch.tensor([[1, 0], [0, 0]], device=device)
    for saved, write in ((state, lambda: reorder_states([state], parents)),
                         (c.k_scale, lambda: kv_cache_append(c, k, k, table, lens)),
                         (c.v_scale, lambda: kv_cache_append(c, k, k, table, lens))):
        w = torch.ones_like(saved, requires_grad=True)
        y, kept = (w * saved).sum(), [(t, t._version) for t in (c.k, c.v)]
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        assert saved is state or all(t._version > v for t, v in kept)
    with torch.inference_mode():  # these have no version to keep
        inside = randn(g, 4, 5).to(device)
        reorder_states([inside], parents)
    want = inside[[0, 1, 2, 2]]
    reorder_states([inside], torch.tensor([[0, 1], [0, 0]], device=device))
    assert torch.equal(inside, want)


@on_devices
def test_tangents_are_refused(device):
    """Forward-mode derivatives would be dropped: refused, as inputs that require a gradient are."""
    import torch.autograd.forward_ad as fwAD
    x, w, scores = torch.randn(4, 128, device=device), torch.ones(128, device=device), torch.zeros(2, 2, device=device)
    cache = alloc_kv_cache(2, 1, 64, 16, device)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device=device), torch.ones(1, dtype=torch.int32, device=device)
    q, parents = x[:1, None, None, :64].to(BF16), torch.zeros(2, 2, dtype=torch.long, device=device)
    with fwAD.dual_level():

        def dual(t):
            return fwAD.make_dual(t, torch.ones_like(t))

        for name, call in (("add_rms_norm_quant", lambda: add_rms_norm_quant(dual(x), w)),
                           ("add_rms_norm_quant", lambda: add_rms_norm_quant(x, dual(w))),
                           ("kv_cache_append", lambda: kv_cache_append(cache, q, dual(q), table, lens)),
                           ("kv_cache_attention", lambda: kv_cache_attention(dual(q), cache, table, lens)),
                           ("beam_select", lambda: beam_select(dual(x), scores)),
                           ("beam_select", lambda: beam_select(x, dual(scores))),
                           ("reorder_states", lambda: reorder_states([dual(x)], parents))):
            with pytest.raises(RuntimeError, match=name + ".*tangent"):
                call()
        with torch.inference_mode():
            add_rms_norm_quant(dual(x), w)
        assert add_rms_norm_quant(fwAD.unpack_dual(dual(x)).primal, w).q.shape == x.shape


@on_devices
def test_negated_views_are_refused(device):
    """A view that negates lazily (the imaginary part of a conjugate) would be read with the other sign."""
    x, w = torch.randn(2, 128, device=device), torch.ones(128, device=device)
    for call in (lambda: add_rms_norm_quant(torch._neg_view(x), w),
                 lambda: beam_select(torch._neg_view(x), torch.zeros(1, 2, device=device))):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    got = add_rms_norm_quant(torch._neg_view(x).resolve_neg(), w)
    assert torch.equal(got.q.float(), add_rms_norm_quant(-x, w).q.float())


# --------------------------------------------------------------------------------------------- together


class Step:
    """A decode step as a server runs it: norm + fp8 projections, append, attention, head, beams, reordered cache."""

    def __init__(self, device, b=2, k=4, vocab=1000, heads=8, kv=2, dim=64, page=16, pages=6):
        from tilelang.ops.fp8_gemm import weight_quant
        g = gen(11)
        n, d = b * k, heads * dim
        self.b, self.k, self.heads, self.kv, self.dim = b, k, heads, kv, dim
        self.embed = randn(g, vocab, d).to(BF16).to(device)
        self.norm_w = torch.ones(d, dtype=BF16, device=device)
        self.wqkv = weight_quant((randn(g, (heads + 2 * kv) * dim, d) * d**-0.5).to(device))
        self.wo = weight_quant((randn(g, d, d) * d**-0.5).to(device))
        # every beam its own pages, so that the pools are states of [beams, pages of one, ...]
        self.cache = alloc_kv_cache(n * pages, kv, dim, page, device)
        self.table = torch.arange(n * pages, dtype=torch.int32, device=device).view(n, pages)
        self.lengths = torch.zeros(n, dtype=torch.int32, device=device)
        self.scores = torch.full((b, k), -math.inf, device=device)
        self.scores[:, 0] = 0.0
        self.tokens = torch.randint(0, vocab, (b, 1), generator=g).repeat_interleave(k, 1).flatten().to(device)
        self.finished = torch.zeros(b, k, dtype=torch.bool, device=device)
        self.states = [t.view(n, pages, -1) for t in self.cache[:4]]

    def __call__(self):
        from tilelang.ops.fp8_gemm import fp8_gemm
        n = self.b * self.k
        self.lengths += 1
        x = self.embed[self.tokens]
        r = add_rms_norm_quant(x, self.norm_w)
        qkv = fp8_gemm(r.q, r.scale, *self.wqkv).view(n, 1, -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv, self.kv], 2)
        kv_cache_append(self.cache, k, v, self.table, self.lengths)
        a = kv_cache_attention(q, self.cache, self.table, self.lengths).view(n, -1)
        r = add_rms_norm_quant(a, self.norm_w, x, return_norm=True)
        h = r.h + fp8_gemm(r.q, r.scale, *self.wo)
        logits = (h.float() @ self.embed.float().t()) * 0.02
        scores, parents, tokens = beam_select(logits, self.scores, finished=self.finished, eos_id=3)
        self.finished.copy_(self.finished.gather(1, parents) | (tokens == 3))
        self.scores.copy_(scores)
        self.tokens.copy_(tokens.flatten())
        reorder_states(self.states, parents)
        return scores, parents, tokens, a


def test_decode_step_cpu():
    step = Step("cpu", b=1, k=2, vocab=64)
    for _ in range(20):
        scores, parents, tokens, a = step()
        assert torch.isfinite(scores).all() and torch.isfinite(a).all()
    assert (scores[:, :-1] >= scores[:, 1:]).all()


@pytest.mark.gpu
def test_decode_step_captured_matches_eager():
    """The step captured into a graph and replayed, with other work in between, against the eager step."""
    eager, graphed = Step("cuda"), Step("cuda")
    first = [t.clone() for t in eager()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for got, want in zip(graphed(), first):  # also the warm-up: another stream than the tensors' own
            assert torch.equal(got, want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed()
    for i in range(40):
        want = [t.clone() for t in eager()]
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
            check_select(torch.randn(2, 3, 777, device="cuda"), torch.zeros(2, 3, device="cuda"), 6)
        for got, ref in zip(out, want):
            assert torch.equal(got, ref), i
    for a, b in zip(eager.cache[:4], graphed.cache[:4]):
        a, b = (t.view(torch.uint8) if t.dtype is FP8 else t for t in (a, b))
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_captured_attentions_do_not_share_scratch():
    """Two graphs of split attention, replayed in turn and at once on two streams."""
    g = gen(12)
    calls = []
    for seed in (1, 2):
        c, table, lens = filled(g, [2500, 1700], 2, 64, 64, "cuda")
        q = randn(gen(seed), 2, 1, 8, 64).to(BF16).cuda()
        calls.append((q, c, table, lens))
    want = [kv_cache_attention(*c) for c in calls]
    graphs, outs = [], []
    for c in calls:
        kv_cache_attention(*c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kv_cache_attention(*c))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref)


@pytest.mark.gpu
def test_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    with torch.cuda.device(0):
        c, table, lens = filled(gen(1), [100], 1, 64, 16, "cuda:1")
        check_attention(torch.randn(1, 1, 2, 64, device="cuda:1").to(BF16), c, table, lens)
        check_select(torch.randn(2, 3, 500, device="cuda:1"), torch.zeros(2, 3, device="cuda:1"))


@pytest.mark.gpu
def test_mixed_devices_are_refused():
    x, w = torch.randn(2, 128, device="cuda").to(BF16), torch.ones(128, dtype=BF16)
    with pytest.raises(ValueError, match="'weight' is on cpu, expected cuda:0"):
        add_rms_norm_quant(x, w)
    with pytest.raises(ValueError, match="'cache.k' is on cpu"):
        c = alloc_kv_cache(1, 1, 64, 16, "cpu")
        t = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
        kv_cache_attention(torch.zeros(1, 1, 1, 64, dtype=BF16, device="cuda"), c, t, t[0])


@on_devices
def test_cache_is_a_plain_tuple(device):
    c = alloc_kv_cache(3, 2, 100, 32, device)
    assert isinstance(c, KVCache) and c.k.shape == (3, 2, 32, 128) and c.v.shape == (3, 2, 128, 32)
    assert c.head_dim == 100 and (c.k_scale == 1).all()
