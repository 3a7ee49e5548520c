"""The feed-forward operators on a GPU against their definitions in 64 bits.

Tolerances, derived from the arithmetic (u = half a step of the element type, 2^-8 for bf16 and 2^-11 for fp16;
e = 2^-24):
  a product       sums of K exact products in fp32; the tensor core may truncate where the formula rounds, so every
                  addition costs at most 2 e of the running magnitude: E(z) = 2 (K + 2) e S with S = sum |x||w| + |b|
  an activation   slopes are at most 1.2, and the fast exponential adds at most 2^-19 of the magnitude: 1.2 E + 2^-19 |.|
  a store         u |value|, and half the smallest step where fp16 ends (2^-25)
  a gradient      dz is stored once more, u |dz|, before the products that read it
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def B(native_lib):
    from flextensor_b200 import backend
    assert backend.lib().ftb_device_check() == 0, "the current device is not sm_100"
    return backend


@pytest.fixture()
def status(B):
    st = B.new_status()
    yield st
    B.check_status(st)


def rand(seed, *shape, scale=1.0, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def act64(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, name):
    z = z.clone().requires_grad_(True)
    return torch.autograd.grad(act64(z, name).sum(), z)[0]


def bounded(got, want, tol, what):
    assert torch.isfinite(want).all()
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its bound (got %s, want %s)" % (
        what, int(bad.sum()), bad.numel(), float((off / tol).max()), got[bad][:4].tolist(), want[bad][:4].tolist())


def store(value, dtype):
    return STEP[dtype] * value.abs() + 2.0 ** -25


def product64(x, w, b):
    """z, and the bound of its fp32 sum."""
    z = x.double() @ w.double().T
    size = x.double().abs() @ w.double().abs().T
    if b is not None:
        z = z + b.double()
        size = size + b.double().abs()
    return z, 2 * (x.shape[1] + 2) * E * size


def forward64(x, w, b, r, act, gated):
    z, ez = product64(x, w, b)
    if gated:
        n = z.shape[1] // 2
        a, u = act64(z[:, :n], act), z[:, n:]
        out = a * u
        tol = (1.2 * ez[:, :n] + 2.0 ** -19 * z[:, :n].abs()) * (u.abs() + ez[:, n:]) + a.abs() * ez[:, n:]
    else:
        out = act64(z, act)
        tol = 1.2 * ez + 2.0 ** -19 * z.abs()
    if r is not None:
        out = out + r.double()
    return out, tol + 4 * E * out.abs(), z, ez


SHAPES = [(1, 128, 64), (1, 333, 1000), (2, 7, 8), (15, 64, 72), (16, 130, 128), (17, 256, 200), (33, 1, 264),
          (64, 129, 512), (65, 300, 136), (127, 640, 64), (128, 128, 128), (129, 513, 192), (257, 384, 1024),
          (300, 1003, 328), (511, 257, 80), (40, 96, 5), (130, 70, 100), (1, 33, 3), (700, 520, 96), (8, 2048, 4096)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("gated", [False, True])
def test_linear(B, status, dtype, t, n, k, gated):
    pick = t + n + k
    act = ACTS[pick % 5]
    wide = 2 * n if gated else n
    x, w = rand(1, t, k, dtype=dtype), rand(2, wide, k, scale=k ** -0.5, dtype=dtype)
    b = rand(3, wide, dtype=dtype) if pick % 2 else None
    r = rand(4, t, n, dtype=dtype) if pick % 3 else None
    z = torch.full((t, wide), 9.0, device="cuda", dtype=dtype) if pick % 4 != 1 else None
    out = torch.full((t, n), float("nan"), device="cuda", dtype=dtype)
    B.linear(x, w, out, bias=b, residual=r, activation=act, gated=gated, preact=z, status=status)
    want, tol, z64, ez = forward64(x, w, b, r, act, gated)
    bounded(out, want, tol + store(want, dtype), "out")
    if z is not None:
        bounded(z, z64, ez + store(z64, dtype), "preact")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
def test_linear_activations(B, status, act, gated):
    """Every activation over a wide range of z (x is a row of ones, so z is the weight)."""
    n = 512
    values = torch.cat([torch.linspace(-30, 30, n), torch.linspace(-3, 3, n)])[: n * (2 if gated else 1)]
    w = torch.zeros(values.numel(), 64)
    w[:, 0] = values
    w = w.to(torch.bfloat16).cuda()
    x = torch.zeros(3, 64, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    out = torch.empty(3, n, device="cuda", dtype=torch.bfloat16)
    B.linear(x, w, out, activation=act, gated=gated, status=status)
    want, tol, _, _ = forward64(x, w, None, None, act, gated)
    bounded(out, want, tol + store(want, torch.bfloat16), act)


def test_linear_residual_in_place(B, status):
    x, w = rand(5, 70, 256), rand(6, 200, 256, scale=1 / 16)
    h = rand(7, 70, 200)
    want, tol, _, _ = forward64(x, w, None, h, "gelu", False)
    B.linear(x, w, h, residual=h, activation="gelu", status=status)
    bounded(h, want, tol + store(want, torch.bfloat16), "in place")


def test_linear_no_tokens(B):
    x, w = rand(1, 0, 64), rand(2, 32, 64)
    out = torch.empty(0, 32, device="cuda", dtype=torch.bfloat16)
    B.linear(x, w, out)
    dw, db = torch.ones_like(w), torch.ones(32, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(B.linear_backward_workspace_bytes(0, 32, 64), dtype=torch.uint8, device="cuda")
    B.linear_backward(x, w, out, dx=torch.empty_like(x), dweight=dw, dbias=db, workspace=ws)
    assert not dw.any() and not db.any()


def test_linear_keeps_rows_of_others_apart(B, status):
    """A token of infinities or NaN reaches its own row only; so does a weight row."""
    x, w = rand(1, 40, 128), rand(2, 150, 128, scale=0.1)
    clean = torch.empty(40, 150, device="cuda", dtype=torch.bfloat16)
    B.linear(x, w, clean, activation="silu", status=status)
    x[3] = float("nan")
    x[17, 5] = float("inf")
    w[140] = float("nan")
    out = torch.empty_like(clean)
    B.linear(x, w, out, activation="silu", status=status)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 17]] = False
    cols = torch.arange(150, device="cuda") != 140
    assert torch.equal(out[keep][:, cols], clean[keep][:, cols])
    assert out[3].isnan().all() and out[:, 140].isnan().all()


def test_linear_refusals(B):
    x, w = rand(1, 4, 64), rand(2, 32, 64)
    out = torch.empty(4, 32, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        B.linear(x, w, out, activation="softplus")
    with pytest.raises(ValueError):
        B.linear(x, w, out, gated=True)               # out would be [4, 16]
    with pytest.raises(TypeError):
        B.linear(x, w.half(), out)
    with pytest.raises(TypeError):
        B.linear(x.float(), w.float(), out.float())
    with pytest.raises(ValueError):
        B.linear(x, rand(2, 64, 32).t(), out)         # not contiguous
    with pytest.raises(ValueError):
        B.linear(x, w, out, bias=rand(3, 31))
    with pytest.raises(ValueError):
        B.linear_backward(x, w, out, dx=torch.empty_like(x), activation="gelu",
                          workspace=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        B.linear_backward(x, w, out, dx=torch.empty_like(x), workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        B.linear_backward(x, w, out, workspace=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    for cfg in ({"tile_n": 48}, {"cluster": 3}, {"split_k": 3}, {"stages": 1}, {"tile_n": 256, "cluster": 1}):
        with pytest.raises(B.FtbError):
            B.linear(x, w, out, cfg=cfg)


# ---------------------------------------------------------------- gradients of a product
def dz64(dy, z, act, gated):
    dy, z = dy.double(), z.double()
    if not gated:
        return dy * (slope64(z, act) if act != "none" else 1)
    n = dy.shape[1]
    return torch.cat([dy * z[:, n:] * slope64(z[:, :n], act), dy * act64(z[:, :n], act)], dim=1)


def gradients64(x, w, dy, z, act, gated):
    dz = dz64(dy, z, act, gated)
    dtype = x.dtype
    size = dy.double().abs()
    if gated:
        n = dy.shape[1]
        size = torch.cat([size * z.double()[:, n:].abs(), size * z.double()[:, :n].abs()], dim=1)
    ed = (0 if act == "none" and not gated else 2.0 ** -18) * size  # fp32 error of dz: slopes of magnitude about 1
    es = ed + (store(dz, dtype) if act != "none" or gated else 0)    # and its store
    full = dz.abs() + es
    n, t = dz.shape[1], dz.shape[0]
    out = {}
    dx = dz @ w.double()
    out["dx"] = (dx, (es + 2 * (n + 2) * E * full) @ w.double().abs() + store(dx, dtype))
    dw = dz.T @ x.double()
    out["dw"] = (dw, (es + 2 * (t + 2) * E * full).T @ x.double().abs() + store(dw, dtype))
    db = dz.sum(0)
    out["db"] = (db, (ed + (t + 70) * E * full).sum(0) + store(db, dtype))
    return out


BACK = [(1, 64, 64), (2, 7, 8), (17, 130, 200), (64, 128, 128), (100, 333, 328), (129, 256, 64), (300, 1003, 136),
        (520, 384, 512), (40, 96, 5), (63, 70, 100), (1025, 72, 264)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k", BACK)
@pytest.mark.parametrize("gated", [False, True])
def test_linear_backward(B, status, dtype, t, n, k, gated):
    act = ACTS[(t + n + k) % 5]
    wide = 2 * n if gated else n
    x, w = rand(1, t, k, dtype=dtype), rand(2, wide, k, scale=0.2, dtype=dtype)
    z, dy = rand(3, t, wide, dtype=dtype), rand(4, t, n, dtype=dtype)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(wide, device="cuda", dtype=dtype)
    ws = torch.full((B.linear_backward_workspace_bytes(t, n, k, gated),), 255, dtype=torch.uint8, device="cuda")
    B.linear_backward(x, w, dy, dx=dx, dweight=dw, dbias=db, preact=z, activation=act, gated=gated, workspace=ws,
                      status=status)
    want = gradients64(x, w, dy, z, act, gated)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        bounded(got, *want[name], name)
    # one at a time gives the same bits
    for name, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
        alone = torch.full_like(got, float("nan"))
        B.linear_backward(x, w, dy, preact=z, activation=act, gated=gated, workspace=ws, status=status, **{name: alone})
        assert torch.equal(alone, got), name


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
def test_linear_backward_against_differences(B, status, act, gated):
    """<gradient, direction> against the central difference of the 64-bit forward along it."""
    t, n, k = 48, 72, 64
    wide = 2 * n if gated else n
    x, w, b = rand(1, t, k, dtype=torch.float16), rand(2, wide, k, scale=0.2, dtype=torch.float16), rand(3, wide, dtype=torch.float16)
    out, z = torch.empty(t, n, device="cuda", dtype=torch.float16), torch.empty(t, wide, device="cuda", dtype=torch.float16)
    B.linear(x, w, out, bias=b, activation=act, gated=gated, preact=z, status=status)
    dy = rand(4, t, n, dtype=torch.float16)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ws = torch.empty(B.linear_backward_workspace_bytes(t, n, k, gated), dtype=torch.uint8, device="cuda")
    B.linear_backward(x, w, dy, dx=dx, dweight=dw, dbias=db, preact=z, activation=act, gated=gated, workspace=ws, status=status)

    def value(x, w, b):
        q = x @ w.T + b
        o = act64(q[:, :n], act) * q[:, n:] if gated else act64(q, act)
        return float((o * dy.double()).sum())

    h = 1e-5
    args = [x.double(), w.double(), b.double()]
    for i, grad in enumerate((dx, dw, db)):
        gen = torch.Generator().manual_seed(10 + i)
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64).cuda()
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + h * v, args[i] - h * v
        slope = (value(*plus) - value(*minus)) / (2 * h)
        # z was rounded to fp16 when it was kept and dz once more: 2^-11 each of terms of the gradient's own size, whose
        # signs are independent; eight standard deviations of the sum, and kinks of relu crossed by that rounding
        terms = (grad.double() * v)
        assert abs(float(terms.sum()) - slope) <= 8 * 2.0 ** -10 * float(terms.square().sum().sqrt()) + 1e-3 * abs(slope) + 0.05, i


# ---------------------------------------------------------------- routing
def scores64(logits, scoring):
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    if scoring == "sigmoid":
        return torch.sigmoid(x)
    p = torch.exp(x - x.max(dim=1, keepdim=True).values)
    p = torch.where(p.isnan(), 0.0, p)
    return torch.where(p > 0, p / p.sum(1, keepdim=True), 0.0)


def route64(logits, top_k, bias, scoring, groups, top_groups, renorm, scale):
    t, e = logits.shape
    s = scores64(logits, scoring)
    c = s + bias.double() if bias is not None else s
    if bias is None and groups == 1:
        c = torch.where(logits.isnan(), -math.inf, logits.double())
    if groups > 1:
        part = c.view(t, groups, -1)
        value = part.sort(dim=2, descending=True).values[:, :, :2].sum(2).clamp(min=-1e200)
        keep = value.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        mask = torch.zeros(t, groups, dtype=torch.bool, device=c.device).scatter_(1, keep, True)
        c = torch.where(mask.repeat_interleave(e // groups, 1), c, torch.nan)
        c = torch.where(c.isnan(), -2e300, c.clamp(min=-1e300))
    ids = c.sort(dim=1, descending=True, stable=True).indices[:, :top_k]
    w = s.gather(1, ids)
    if renorm:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return ids.to(torch.int32), w * scale


ROUTES = [(1, 8, 2, 1, 1), (3, 5, 5, 1, 1), (16, 64, 6, 1, 1), (7, 33, 4, 1, 1), (50, 128, 8, 4, 2), (41, 256, 8, 8, 4),
          (9, 60, 6, 4, 2), (5, 96, 3, 32, 5), (130, 512, 10, 1, 1), (6, 1024, 32, 16, 3), (33, 24, 8, 2, 1), (4, 1, 1, 1, 1),
          (20, 8, 3, 8, 5), (11, 1000, 7, 10, 4)]


@pytest.mark.parametrize("t,e,k,groups,top_groups", ROUTES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route(B, t, e, k, groups, top_groups, scoring, dtype):
    logits = rand(t + e, t, e, scale=2.0, dtype=dtype)
    for bias in (None, rand(e, e, scale=0.1, dtype=torch.float32)):
        for renorm, scale in ((True, 1.0), (False, 2.5)):
            ids = torch.full((t, k), -7, device="cuda", dtype=torch.int32)
            weights = torch.full((t, k), float("nan"), device="cuda")
            B.route_experts(logits, ids, weights, bias=bias, scoring=scoring, groups=groups, top_groups=top_groups,
                            renormalize=renorm, scale=scale)
            want_ids, want = route64(logits, k, bias, scoring, groups, top_groups, renorm, scale)
            assert torch.equal(ids, want_ids)
            # exp, reciprocals and a sum of e terms in fp32, each a few steps
            bounded(weights, want, (32 + e / 8) * E * want.abs() + 1e-37, "weights")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_near_ties(B, scoring, groups, top_groups):
    """Rows whose scores plus bias agree to a few units of 2^-24 or exactly: 64 bits decide, then the index."""
    t, e, k = 64, 32, 6
    gen = torch.Generator().manual_seed(3)
    logits = torch.randn(t, 1, generator=gen).expand(t, e).clone()
    logits[: t // 2] += torch.randint(-2, 3, (t // 2, e), generator=gen) * 2.0 ** -22
    bias = torch.zeros(e)
    bias[torch.randperm(e, generator=gen)[: e // 2]] = 2.0 ** -23
    logits, bias = logits.cuda(), bias.cuda()
    for b in (bias, None):
        ids, weights = torch.empty(t, k, device="cuda", dtype=torch.int32), torch.empty(t, k, device="cuda")
        B.route_experts(logits, ids, weights, bias=b, scoring=scoring, groups=groups, top_groups=top_groups)
        want_ids, want = route64(logits, k, b, scoring, groups, top_groups, True, 1.0)
        # equal logits give equal scores on both sides; unequal ones differ by 2^-24 of a score, far above 2^-53
        assert torch.equal(ids, want_ids)
        bounded(weights, want, 64 * E * want.abs(), "weights")


@pytest.mark.parametrize("e,k,groups,top_groups", [(64, 6, 1, 1), (256, 8, 8, 4), (60, 5, 4, 2), (100, 9, 1, 1), (32, 4, 32, 6)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_bias_disables_experts(B, e, k, groups, top_groups, scoring):
    """A bias of -inf: the expert is taken only when no other is left."""
    t = 40
    logits, bias = rand(e, t, e, dtype=torch.float32), rand(1, e, scale=0.1, dtype=torch.float32)
    bias[::3] = -math.inf
    bias[e // 2:e // 2 + 4] = -math.inf
    ids, weights = torch.empty(t, k, device="cuda", dtype=torch.int32), torch.empty(t, k, device="cuda")
    B.route_experts(logits, ids, weights, bias=bias, scoring=scoring, groups=groups, top_groups=top_groups, renormalize=False)
    want_ids, want = route64(logits, k, bias, scoring, groups, top_groups, False, 1.0)
    assert torch.equal(ids, want_ids)
    bounded(weights, want, (32 + e / 8) * E * want.abs() + 1e-37, "weights")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_masked_rows(B, scoring, dtype):
    t, e, k = 8, 40, 4
    logits = rand(1, t, e, dtype=dtype)
    low = torch.finfo(dtype).min
    logits[0, 3:] = -math.inf        # fewer experts left than wanted
    logits[1] = -math.inf            # none left
    logits[2, ::2] = float("nan")
    logits[3] = low                  # the type's lowest value everywhere
    logits[4, 5:] = low
    logits[5, 7] = math.inf
    logits[6] = float("nan")
    logits[7] = -200.0               # every sigmoid underflows
    for renorm in (True, False):
        ids, weights = torch.empty(t, k, device="cuda", dtype=torch.int32), torch.empty(t, k, device="cuda")
        B.route_experts(logits, ids, weights, scoring=scoring, renormalize=renorm)
        assert torch.isfinite(weights).all()
        assert ids[1].tolist() == ids[6].tolist() == ids[3].tolist() == ids[7].tolist() == [0, 1, 2, 3]
        assert ids[0].tolist()[3] == 3 and weights[0, 3] == 0
        assert not weights[1].any() and not weights[6].any()
        assert ids[5, 0] == 7 and not (ids[2] % 2 == 0).any()
        assert ids[4].sort().values.tolist()[:1] != [5]
        if renorm:
            rows = [0, 2, 5, 7] + ([3] if scoring == "softmax" else [])
            assert torch.allclose(weights[rows].sum(1), torch.ones(len(rows), device="cuda"), atol=1e-6)
            assert torch.allclose(weights[7], torch.full((k,), 0.25, device="cuda"), atol=1e-6)
        back = torch.full_like(logits, float("nan"))
        B.route_experts_backward(logits, ids, torch.ones(t, k, device="cuda"), back, scoring=scoring, renormalize=renorm)
        assert torch.isfinite(back.float()).all()


@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (16, 64, 6), (7, 33, 4), (130, 128, 8), (5, 1000, 32), (3, 1, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route_backward(B, t, e, k, scoring, renorm, dtype):
    logits = rand(t + e, t, e, scale=1.5, dtype=dtype)
    gen = torch.Generator().manual_seed(2)
    ids = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)]).to(torch.int32).cuda()
    if k > 1:
        ids[0, 1] = ids[0, 0]                 # the same expert twice
        ids[t // 2, 0] = -1                   # dropped
        ids[t - 1, 1] = e
    dweights = rand(5, t, k, dtype=torch.float32)
    got = torch.full_like(logits, float("nan"))
    B.route_experts_backward(logits, ids, dweights, got, scoring=scoring, renormalize=renorm, scale=1.7)
    x = logits.double().requires_grad_(True)
    s = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    live = (ids >= 0) & (ids < e)
    w = s.gather(1, torch.where(live, ids, 0).long()) * live
    if renorm:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(live.any(1, keepdim=True), total, 1.0)  # a row without any valid id has no gradient
    want = torch.autograd.grad((w * 1.7 * dweights * live).sum(), x)[0]
    # terms of the row's largest size meet and may cancel: a few steps of that size, times the sum over e
    size = (dweights.double().abs() * 1.7).amax(1, keepdim=True) * (s if not renorm else 1)
    bounded(got, want, (64 + e / 4) * E * size + store(want, dtype) + 1e-30, "dlogits")


# ---------------------------------------------------------------- experts
def make_ids(t, k, e, drop=0.0, skew=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    wish = torch.randn(t, e, generator=gen) + skew * torch.randn(e, generator=gen)
    ids = wish.topk(k, dim=1).indices.to(torch.int32)
    if drop:
        ids[torch.rand(t, k, generator=gen) < drop] = -1
    return ids.cuda()


def plan64(ids, e):
    flat = ids.flatten().cpu().tolist()
    rows = [[] for _ in range(e)]
    for r, i in enumerate(flat):
        if 0 <= i < e:
            rows[i].append(r)
    order = [r for one in rows for r in one]
    offsets = [0]
    for one in rows:
        offsets.append(offsets[-1] + len(one))
    slots = [-1] * len(flat)
    for p, r in enumerate(order):
        slots[r] = p
    return offsets, order + [-1] * (len(flat) - len(order)), slots


def planned(B, ids, e):
    plan = B.ExpertPlan(ids.shape[0], ids.shape[1], e)
    B.expert_plan(ids, plan)
    return plan


@pytest.mark.parametrize("t,k,e,drop", [(1, 1, 1, 0), (1, 8, 64, 0), (16, 4, 8, 0.3), (100, 2, 33, 0), (700, 6, 1024, 0.1),
                                        (1500, 4, 40, 0.05), (5000, 8, 256, 0), (8, 32, 32, 0), (3000, 3, 5, 1.0)])
def test_expert_plan(B, t, k, e, drop):
    ids = make_ids(t, k, e, drop, seed=t)
    if t > 10:
        ids[1, 0], ids[2, 0] = e, 2 ** 31 - 1
    plan = planned(B, ids, e)
    offsets, order, slots = plan64(ids, e)
    assert plan.offsets.tolist() == offsets and plan.order.tolist() == order and plan.slots.tolist() == slots
    B.expert_plan(torch.zeros_like(ids), plan)  # one expert takes all; the buffers hold another plan
    assert plan.offsets.tolist() == [0] + [t * k] * e and plan.order.tolist() == list(range(t * k))


def test_expert_plan_empty(B):
    plan = B.ExpertPlan(0, 2, 7)
    plan.offsets.fill_(5)
    B.expert_plan(torch.empty(0, 2, device="cuda", dtype=torch.int32), plan)
    assert plan.offsets.tolist() == [0] * 8
    w = rand(1, 7, 32, 64)
    out = torch.empty(0, 32, device="cuda", dtype=torch.bfloat16)
    B.expert_linear(rand(1, 0, 64), w, plan, out)
    dw, db = torch.ones_like(w), torch.ones(7, 32, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(B.expert_linear_backward_workspace_bytes(plan, 32, 64), dtype=torch.uint8, device="cuda")
    B.expert_linear_backward(rand(1, 0, 64), w, plan, out, dweight=dw, dbias=db, workspace=ws)
    assert not dw.any() and not db.any()


EXPERTS = [(1, 1, 1, 64, 64), (1, 8, 64, 130, 128), (3, 2, 4, 7, 8), (16, 4, 8, 256, 200), (100, 2, 5, 300, 136),
           (257, 3, 6, 129, 64), (40, 6, 128, 64, 72), (600, 2, 3, 512, 264), (50, 2, 4, 33, 20), (2000, 1, 9, 96, 96), (3, 32, 1024, 40, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,e,n,width", EXPERTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_expert_linear(B, status, dtype, t, k, e, n, width, gated, gather):
    pick = t + n + width
    act = ACTS[pick % 5]
    wide = 2 * n if gated else n
    ids = make_ids(t, k, e, drop=0.15 if pick % 2 else 0.0, seed=pick)
    plan = planned(B, ids, e)
    rows = t * k
    x = rand(1, t if gather else rows, width, dtype=dtype)
    w = rand(2, e, wide, width, scale=width ** -0.5, dtype=dtype)
    b = rand(3, e, wide, dtype=dtype) if pick % 3 else None
    out = torch.full((rows, n), 7.0, device="cuda", dtype=dtype)
    z = torch.full((rows, wide), 7.0, device="cuda", dtype=dtype) if pick % 4 != 1 else None
    offsets, order, _ = plan64(ids, e)
    used = offsets[-1]
    if not gather:
        x[used:] = float("nan")  # nothing reads the rows behind the last place into a result
    B.expert_linear(x, w, plan, out, bias=b, activation=act, gated=gated, gather=gather, preact=z, status=status)
    place = torch.tensor(order[:used], device="cuda", dtype=torch.long)
    src = x[place // k] if gather else x[:used]
    assert (out[used:] == 7).all() and (z is None or (z[used:] == 7).all())
    for i in range(e):
        a, c = offsets[i], offsets[i + 1]
        if a == c:
            continue
        want, tol, z64, ez = forward64(src[a:c], w[i], b[i] if b is not None else None, None, act, gated)
        bounded(out[a:c], want, tol + store(want, dtype), "out of expert %d" % i)
        if z is not None:
            bounded(z[a:c], z64, ez + store(z64, dtype), "preact of expert %d" % i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,e,n,width", EXPERTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_expert_linear_backward(B, status, dtype, t, k, e, n, width, gated, gather):
    pick = t + n + width
    act = ACTS[(pick + 1) % 5]
    wide = 2 * n if gated else n
    ids = make_ids(t, k, e, drop=0.15 if pick % 2 else 0.0, seed=pick)
    plan = planned(B, ids, e)
    rows = t * k
    x = rand(1, t if gather else rows, width, dtype=dtype)
    w = rand(2, e, wide, width, scale=0.2, dtype=dtype)
    z, dy = rand(3, rows, wide, dtype=dtype), rand(4, rows, n, dtype=dtype)
    offsets, order, _ = plan64(ids, e)
    used = offsets[-1]
    for one in (z, dy) + (() if gather else (x,)):
        one[used:] = float("nan")  # rows behind the last place
    dx = torch.full((rows, width), 7.0, device="cuda", dtype=dtype)
    dw, db = torch.full_like(w, float("nan")), torch.full((e, wide), float("nan"), device="cuda", dtype=dtype)
    ws = torch.full((B.expert_linear_backward_workspace_bytes(plan, n, width, gated),), 255, dtype=torch.uint8, device="cuda")
    B.expert_linear_backward(x, w, plan, dy, dx=dx, dweight=dw, dbias=db, preact=z, activation=act, gated=gated,
                             gather=gather, workspace=ws, status=status)
    place = torch.tensor(order[:used], device="cuda", dtype=torch.long)
    src = x[place // k] if gather else x[:used]
    assert (dx[used:] == 7).all()
    for i in range(e):
        a, c = offsets[i], offsets[i + 1]
        if a == c:
            assert not dw[i].any() and not db[i].any()
            continue
        want = gradients64(src[a:c], w[i], dy[a:c], z[a:c], act, gated)
        for name, got in (("dx", dx[a:c]), ("dw", dw[i]), ("db", db[i])):
            bounded(got, *want[name], "%s of expert %d" % (name, i))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,e,n", [(1, 1, 1, 8), (5, 3, 4, 77), (33, 8, 16, 1024), (200, 2, 6, 1032), (9, 32, 40, 6)])
@pytest.mark.parametrize("plain", [False, True])
def test_expert_combine(B, dtype, t, k, e, n, plain):
    ids = make_ids(t, k, e, drop=0.2, seed=t)
    ids[0] = -1  # a token without any row
    plan = planned(B, ids, e)
    used = int(plan.offsets[-1])
    y = rand(1, t * k, n, dtype=dtype)
    y[used:] = float("nan")
    weights = None if plain else torch.rand(t, k, device="cuda")
    residual = None if plain else rand(2, t, n, dtype=dtype)
    out = torch.full((t, n), float("nan"), device="cuda", dtype=dtype)
    B.expert_combine(y, plan, out, weights=weights, residual=residual)
    slots = plan.slots.view(t, k).long()
    live = (slots >= 0)[:, :, None]
    part = torch.where(live, y.double()[slots.clamp(min=0)], 0.0)
    w64 = torch.ones(t, k, 1, device="cuda", dtype=torch.float64) if plain else weights.double()[:, :, None]
    want = (part * w64).sum(1) + (0 if plain else residual.double())
    size = (part * w64).abs().sum(1) + (0 if plain else residual.double().abs())
    bounded(out, want, 2 * (k + 1) * E * size + store(want, dtype), "out")
    if not plain:
        B.expert_combine(y, plan, residual, weights=weights, residual=residual)  # in place
        assert torch.equal(residual, out)
    # gradients
    dout = rand(3, t, n, dtype=dtype)
    dy, dweights = torch.full_like(y, 7.0), torch.full((t, k), float("nan"), device="cuda")
    B.expert_combine_backward(dout, plan, y=y, weights=weights, dy=dy, dweights=dweights)
    assert (dy[used:] == 7).all()
    order = plan.order[:used].long()
    want_dy = dout.double()[order // k] * (1 if plain else weights.double().flatten()[order][:, None])
    bounded(dy[:used], want_dy, E * want_dy.abs() + store(want_dy, dtype), "dy")
    terms = part * dout.double()[:, None, :]
    bounded(dweights, terms.sum(2), 2 * (n + 2) * E * terms.abs().sum(2) + 1e-30, "dweights")
    alone = torch.empty_like(dweights)
    B.expert_combine_backward(dout, plan, y=y, weights=weights, dweights=alone)
    assert torch.equal(alone, dweights)


def test_expert_refusals(B):
    ids = make_ids(6, 2, 4)
    plan = planned(B, ids, 4)
    x, w = rand(1, 12, 64), rand(2, 4, 32, 64)
    out = torch.empty(12, 32, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        B.expert_linear(x, w, plan, out, gather=True)     # x has a row per place, not per token
    with pytest.raises(ValueError):
        B.expert_linear(x, rand(2, 5, 32, 64), plan, out)
    with pytest.raises(ValueError):
        B.expert_linear(x, rand(2, 4, 31, 64), plan, out, gated=True)
    with pytest.raises(TypeError):
        B.expert_linear(x, w, plan.offsets, out)
    with pytest.raises(TypeError):
        B.expert_plan(ids.long(), plan)
    with pytest.raises(ValueError):
        B.expert_plan(ids[:5], plan)
    with pytest.raises(ValueError):
        B.ExpertPlan(4, 33, 64)
    with pytest.raises(ValueError):
        B.ExpertPlan(4, 2, 1025)
    with pytest.raises(B.FtbError):
        B.expert_linear(x, w, plan, out, cfg={"split_k": 2})
    logits, weights = rand(1, 6, 4, dtype=torch.float32), torch.empty(6, 2, device="cuda")
    with pytest.raises(ValueError):
        B.route_experts(logits, ids, weights, groups=3)
    with pytest.raises(ValueError):
        B.route_experts(logits, torch.empty(6, 5, device="cuda", dtype=torch.int32), torch.empty(6, 5, device="cuda"))
    with pytest.raises(ValueError):
        B.route_experts(logits, ids, weights, scoring="relu")
    with pytest.raises(TypeError):
        B.route_experts(logits, ids.long(), weights)
    with pytest.raises(ValueError):
        B.expert_combine_backward(torch.empty(6, 32, device="cuda", dtype=torch.bfloat16), plan)
    with pytest.raises(ValueError):
        B.expert_combine_backward(torch.empty(6, 32, device="cuda", dtype=torch.bfloat16), plan,
                                  dweights=torch.empty(6, 2, device="cuda"))


# ---------------------------------------------------------------- every variant of the tensor-core kernel
CFGS = [{"tile_n": 16}, {"tile_n": 32}, {"tile_n": 64, "split_k": 1}, {"tile_n": 128}, {"cluster": 2, "tile_n": 128},
        {"cluster": 2, "tile_n": 256}, {"tile_n": 16, "split_k": 2}, {"tile_n": 32, "split_k": 4}, {"tile_n": 64, "split_k": 8},
        {"stages": 2}, {"tile_n": 64, "stages": 2, "split_k": 8}, {"cluster": 2}, {"split_k": 4}]


@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: "-".join("%s%d" % i for i in c.items()))
@pytest.mark.parametrize("gated", [False, True])
def test_linear_knobs(B, status, cfg, gated):
    for t, n, k in ((1, 130, 264), (75, 200, 520), (300, 700, 200)):
        x, w = rand(1, t, k), rand(2, n * (2 if gated else 1), k, scale=k ** -0.5)
        b, r = rand(3, w.shape[0]), rand(4, t, n)
        out = torch.full((t, n), float("nan"), device="cuda", dtype=torch.bfloat16)
        B.linear(x, w, out, bias=b, residual=r, activation="gelu_tanh", gated=gated, cfg=cfg, status=status)
        want, tol, _, _ = forward64(x, w, b, r, "gelu_tanh", gated)
        bounded(out, want, tol + store(want, torch.bfloat16), "%s %s" % (cfg, (t, n, k)))
        again = torch.empty_like(out)
        B.linear(x, w, again, bias=b, residual=r, activation="gelu_tanh", gated=gated, cfg=cfg, status=status)
        assert torch.equal(out, again)  # no order of sums depends on timing


@pytest.mark.parametrize("cfg", [c for c in CFGS if c.get("split_k", 1) == 1], ids=lambda c: "-".join("%s%d" % i for i in c.items()))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_expert_linear_knobs(B, status, cfg, gated, gather):
    t, k, e, n, width = 210, 3, 5, 330, 200
    ids = make_ids(t, k, e, drop=0.1)
    plan = planned(B, ids, e)
    offsets, order, _ = plan64(ids, e)
    x, w = rand(1, t if gather else t * k, width), rand(2, e, n * (2 if gated else 1), width, scale=width ** -0.5)
    out = torch.full((t * k, n), 7.0, device="cuda", dtype=torch.bfloat16)
    B.expert_linear(x, w, plan, out, activation="silu", gated=gated, gather=gather, cfg=cfg, status=status)
    used = offsets[-1]
    src = x[torch.tensor(order[:used], device="cuda") // k] if gather else x[:used]
    for i in range(e):
        a, c = offsets[i], offsets[i + 1]
        want, tol, _, _ = forward64(src[a:c], w[i], None, None, "silu", gated)
        bounded(out[a:c], want, tol + store(want, torch.bfloat16), "expert %d" % i)
    assert (out[used:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k,gated", [(1300, 2600, 136, False), (1025, 1111, 72, True), (520, 6000, 64, False), (2100, 600, 328, True)])
def test_linear_large(B, status, dtype, t, n, k, gated):
    """Sizes whose defaults are the pair tiles, forward and backward."""
    wide = 2 * n if gated else n
    x, w, b = rand(1, t, k, dtype=dtype), rand(2, wide, k, scale=k ** -0.5, dtype=dtype), rand(3, wide, dtype=dtype)
    out, z = torch.empty(t, n, device="cuda", dtype=dtype), torch.empty(t, wide, device="cuda", dtype=dtype)
    B.linear(x, w, out, bias=b, activation="silu", gated=gated, preact=z, status=status)
    want, tol, z64, ez = forward64(x, w, b, None, "silu", gated)
    bounded(out, want, tol + store(want, dtype), "out")
    bounded(z, z64, ez + store(z64, dtype), "preact")
    dy = rand(4, t, n, dtype=dtype)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ws = torch.empty(B.linear_backward_workspace_bytes(t, n, k, gated), dtype=torch.uint8, device="cuda")
    B.linear_backward(x, w, dy, dx=dx, dweight=dw, dbias=db, preact=z, activation="silu", gated=gated, workspace=ws, status=status)
    want = gradients64(x, w, dy, z, "silu", gated)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        bounded(got, *want[name], name)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_expert_large(B, status, gather, gated):
    """Groups long enough for the pair tiles, one of them empty and one of a single row."""
    t, k, e, n, width = 1700, 2, 4, 1300, 520
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 2, (t, k), generator=gen, dtype=torch.int32)
    ids[5, 0] = 3
    ids[-40:] = -1
    ids = ids.cuda()
    plan = planned(B, ids, e)
    offsets, order, _ = plan64(ids, e)
    used, rows, wide = offsets[-1], t * k, n * (2 if gated else 1)
    x, w = rand(1, t if gather else rows, width), rand(2, e, wide, width, scale=width ** -0.5)
    out, z = torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16), torch.zeros(rows, wide, device="cuda", dtype=torch.bfloat16)
    B.expert_linear(x, w, plan, out, activation="gelu", gated=gated, gather=gather, preact=z, status=status)
    src = x[torch.tensor(order[:used], device="cuda") // k] if gather else x[:used]
    dy = rand(3, rows, n)
    dx, dw, db = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16), torch.empty_like(w), torch.empty(e, wide, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(B.expert_linear_backward_workspace_bytes(plan, n, width, gated), dtype=torch.uint8, device="cuda")
    B.expert_linear_backward(x, w, plan, dy, dx=dx, dweight=dw, dbias=db, preact=z, activation="gelu", gated=gated, gather=gather,
                             workspace=ws, status=status)
    for i in range(e):
        a, c = offsets[i], offsets[i + 1]
        if a == c:
            assert not dw[i].any() and not db[i].any()
            continue
        want, tol, z64, ez = forward64(src[a:c], w[i], None, None, "gelu", gated)
        bounded(out[a:c], want, tol + store(want, torch.bfloat16), "out %d" % i)
        bounded(z[a:c], z64, ez + store(z64, torch.bfloat16), "preact %d" % i)
        want = gradients64(src[a:c], w[i], dy[a:c], z[a:c], "gelu", gated)
        for name, got in (("dx", dx[a:c]), ("dw", dw[i]), ("db", db[i])):
            bounded(got, *want[name], "%s %d" % (name, i))
    assert not out[used:].any() and not dx[used:].any()


def shifted(t, by=1):
    """The same values in a contiguous tensor whose base is ``by`` elements off a 16-byte boundary."""
    flat = torch.empty(t.numel() + 16, device="cuda", dtype=t.dtype)
    view = flat[by:by + t.numel()].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("which", range(6))
def test_unaligned_bases(B, status, which):
    """Any one operand, or all of them, off a 16-byte boundary: other accesses, the same values within their bounds."""
    t, n, k = 70, 136, 128
    x, w, b, r, dy = rand(1, t, k), rand(2, 2 * n, k, scale=0.1), rand(3, 2 * n), rand(4, t, n), rand(5, t, n)
    move = lambda i, v: shifted(v) if which in (i, 5) else v
    x, w, r, dy = move(0, x), move(1, w), move(2, r), move(4, dy)
    out, z = move(3, torch.empty_like(r)), move(4, torch.empty(t, 2 * n, device="cuda", dtype=torch.bfloat16))
    B.linear(x, w, out, bias=move(2, b), residual=r, activation="silu", gated=True, preact=z, status=status)
    want, tol, z64, ez = forward64(x, w, b, r, "silu", True)
    bounded(out, want, tol + store(want, torch.bfloat16), "out")
    bounded(z, z64, ez + store(z64, torch.bfloat16), "preact")
    dx, dw, db = move(0, torch.empty_like(x)), move(1, torch.empty_like(w)), move(2, torch.empty_like(b))
    ws = torch.empty(B.linear_backward_workspace_bytes(t, n, k, True), dtype=torch.uint8, device="cuda")
    B.linear_backward(x, w, dy, dx=dx, dweight=dw, dbias=db, preact=z, activation="silu", gated=True, workspace=ws, status=status)
    want = gradients64(x, w, dy, z, "silu", True)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        bounded(got, *want[name], name)
    logits = move(0, rand(6, t, 64, dtype=torch.float32))
    bias = move(1, rand(7, 64, dtype=torch.float32))
    ids, weights = torch.empty(t, 4, device="cuda", dtype=torch.int32), torch.empty(t, 4, device="cuda")
    B.route_experts(logits, ids, weights, bias=bias, scoring="sigmoid", groups=4, top_groups=2)
    assert torch.equal(ids, route64(logits, 4, bias, "sigmoid", 4, 2, True, 1.0)[0])
    plan = planned(B, ids, 64)
    y = move(3, rand(8, t * 4, n))
    got = move(4, torch.empty(t, n, device="cuda", dtype=torch.bfloat16))
    B.expert_combine(y, plan, got, weights=weights)
    part = y.double()[plan.slots.long()].view(t, 4, n) * weights.double()[:, :, None]
    bounded(got, part.sum(1), 10 * E * part.abs().sum(1) + store(part.sum(1), torch.bfloat16), "combine")


def test_every_row_dropped(B, status):
    t, k, e, n, width = 20, 3, 5, 72, 64
    plan = planned(B, torch.full((t, k), -1, device="cuda", dtype=torch.int32), e)
    assert plan.offsets.tolist() == [0] * 6 and (plan.order == -1).all() and (plan.slots == -1).all()
    nan = lambda *s: torch.full(s, float("nan"), device="cuda", dtype=torch.bfloat16)
    w = rand(1, e, n, width)
    out, dx = torch.full((t * k, n), 7.0, device="cuda", dtype=torch.bfloat16), torch.full((t * k, width), 7.0, device="cuda", dtype=torch.bfloat16)
    for gather in (False, True):
        x = nan(t if gather else t * k, width)
        B.expert_linear(x, w, plan, out, gather=gather, status=status)
        dw, db = nan(e, n, width), nan(e, n)
        ws = torch.empty(B.expert_linear_backward_workspace_bytes(plan, n, width), dtype=torch.uint8, device="cuda")
        B.expert_linear_backward(x, w, plan, nan(t * k, n), dx=dx, dweight=dw, dbias=db, gather=gather, workspace=ws, status=status)
        assert not dw.any() and not db.any()
    assert (out == 7).all() and (dx == 7).all()
    r = rand(2, t, n)
    total, dweights = nan(t, n), torch.full((t, k), float("nan"), device="cuda")
    B.expert_combine(nan(t * k, n), plan, total, weights=torch.rand(t, k, device="cuda"), residual=r)
    assert torch.equal(total, r)
    B.expert_combine_backward(r, plan, y=nan(t * k, n), dweights=dweights)
    assert not dweights.any()


def test_no_tokens_anywhere(B):
    new = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
    logits, ids, weights = new(0, 8, dtype=torch.float32), new(0, 2, dtype=torch.int32), new(0, 2, dtype=torch.float32)
    B.route_experts(logits, ids, weights, groups=2, top_groups=1)
    B.route_experts_backward(logits, ids, weights, logits)
    plan = planned(B, ids, 8)
    y, out = new(0, 24), new(0, 24)
    B.expert_combine(y, plan, out, weights=weights)
    B.expert_combine_backward(out, plan, y=y, dy=y, dweights=weights)
    assert plan.offsets.tolist() == [0] * 9
    w = rand(1, 8, 24, 16)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    for gather in (False, True):
        dw, db = torch.ones_like(w), torch.ones(8, 24, device="cuda", dtype=torch.bfloat16)
        B.expert_linear(new(0, 16), w, plan, y, gather=gather)
        B.expert_linear_backward(new(0, 16), w, plan, y, dx=new(0, 16), gather=gather, workspace=ws)
        B.expert_linear_backward(new(0, 16), w, plan, y, dweight=dw, dbias=db, gather=gather, workspace=ws)
        assert not dw.any() and not db.any()
    B.linear_backward(new(0, 16), w[0], y, dx=new(0, 16), workspace=ws)
    B.linear_backward(new(0, 16), w[0], y, dx=new(0, 16), preact=y, activation="gelu", workspace=ws)


def test_the_same_expert_twice(B, status):
    """A token that names one expert in two slots has two rows there; both count."""
    t, n, width = 10, 40, 64
    ids = torch.tensor([[1, 1, 0]] * t, dtype=torch.int32, device="cuda")
    plan = planned(B, ids, 3)
    x, w = rand(1, t, width), rand(2, 3, n, width, scale=0.125)
    y, out = torch.empty(3 * t, n, device="cuda", dtype=torch.bfloat16), torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    B.expert_linear(x, w, plan, y, gather=True, status=status)
    weights = torch.tensor([[0.5, 0.25, 2.0]] * t, device="cuda")
    B.expert_combine(y, plan, out, weights=weights)
    want = 0.75 * (x.double() @ w[1].double().T) + 2.0 * (x.double() @ w[0].double().T)
    size = 0.75 * (x.double().abs() @ w[1].double().abs().T) + 2.0 * (x.double().abs() @ w[0].double().abs().T)
    # every row is stored once on the way: 2^-8 of each, and the sums of both steps
    rows = 0.75 * (x.double() @ w[1].double().T).abs() + 2.0 * (x.double() @ w[0].double().T).abs()
    bounded(out, want, 2.0 ** -8 * rows + 2 * (width + 6) * E * size + store(want, torch.bfloat16), "out")


def test_results_past_32_bits(B, status):
    """An output of 2.3e9 elements: the last rows lie behind 2^31 of them."""
    t, n, k = 70000, 33000, 64
    x, w = rand(1, t, k), rand(2, n, k, scale=0.1)
    out = torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    B.linear(x, w, out, activation="relu", status=status)
    rows = [0, 1, 65000, 65077, t - 2, t - 1]  # 2^31 / 33000 = 65075.3
    want, tol, _, _ = forward64(x[rows], w, None, None, "relu", False)
    bounded(out[rows], want, tol + store(want, torch.bfloat16), "rows")
    del out
    # the same behind the sorted places of two experts
    plan = planned(B, (torch.arange(t, device="cuda") >= 40000).to(torch.int32)[:, None].contiguous(), 2)
    w2 = rand(3, 2, n, k, scale=0.1)
    out = torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    B.expert_linear(x, w2, plan, out, status=status)
    for i, one in ((0, [0, 39999]), (1, [40000, 65077, t - 1])):
        want, tol, _, _ = forward64(x[one], w2[i], None, None, "none", False)
        bounded(out[one], want, tol + store(want, torch.bfloat16), "expert %d" % i)
    dx = torch.empty_like(x)
    ws = torch.empty(B.expert_linear_backward_workspace_bytes(plan, n, k), dtype=torch.uint8, device="cuda")
    B.expert_linear_backward(x, w2, plan, out, dx=dx, workspace=ws, status=status)
    for i, one in ((0, [0, 39999]), (1, [40000, 65077, t - 1])):
        dy = out[one].double()
        want = dy @ w2[i].double()
        bounded(dx[one], want, 2 * (n + 2) * E * (dy.abs() @ w2[i].double().abs()) + store(want, torch.bfloat16), "dx")


# ---------------------------------------------------------------- together, as a model uses them
class Block(object):
    """A mixture-of-experts feed-forward block with a shared expert, forward and backward, on buffers of its own."""

    def __init__(self, B, t=90, k=2, e=6, d=256, h=136, seed=0):
        self.B, self.t, self.k, self.e, self.d, self.h = B, t, k, e, d, h
        new = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
        self.x, self.dout = rand(seed, t, d), rand(seed + 1, t, d)
        self.router = rand(seed + 2, 1, e, d, scale=d ** -0.5)
        self.w1, self.w2 = rand(seed + 3, e, 2 * h, d, scale=d ** -0.5), rand(seed + 4, e, d, h, scale=h ** -0.5)
        self.s1, self.s2 = rand(seed + 5, 2 * h, d, scale=d ** -0.5), rand(seed + 6, d, h, scale=h ** -0.5)
        self.bias = rand(seed + 7, e, scale=0.05, dtype=torch.float32)
        self.logits, self.ids, self.weights = new(1, t, e, dtype=torch.float32), new(t, k, dtype=torch.int32), new(t, k, dtype=torch.float32)
        self.plan = B.ExpertPlan(t, k, e)
        r = t * k
        self.z1, self.a1, self.y = new(r, 2 * h), new(r, h), new(r, d)
        self.zs, self.as_, self.shared, self.out = new(t, 2 * h), new(t, h), new(t, d), new(t, d)
        self.dy, self.da, self.dz = new(r, d), new(r, h), new(r, d)
        self.dw2, self.dw1, self.ds1, self.ds2 = new(e, d, h), new(e, 2 * h, d), new(2 * h, d), new(d, h)
        self.dweights, self.dlogits, self.dx, self.das = new(t, k, dtype=torch.float32), new(t, e, dtype=torch.float32), new(t, d), new(t, h)
        byte = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")
        self.ws = byte(max(B.expert_linear_backward_workspace_bytes(self.plan, h, d, True),
                           B.expert_linear_backward_workspace_bytes(self.plan, d, h),
                           B.linear_backward_workspace_bytes(t, h, d, True), B.linear_backward_workspace_bytes(t, d, h)))
        self.status = B.new_status()

    def run(self):
        B, st = self.B, self.status
        B.bgemm_bf16(self.x[None], self.router, self.logits, trans_b=True, status=st)
        logits = self.logits[0]
        B.route_experts(logits, self.ids, self.weights, bias=self.bias, scoring="sigmoid")
        B.expert_plan(self.ids, self.plan)
        B.linear(self.x, self.s1, self.as_, activation="silu", gated=True, preact=self.zs, status=st)
        B.linear(self.as_, self.s2, self.shared, residual=self.x, status=st)
        B.expert_linear(self.x, self.w1, self.plan, self.a1, activation="silu", gated=True, gather=True, preact=self.z1, status=st)
        B.expert_linear(self.a1, self.w2, self.plan, self.y, status=st)
        B.expert_combine(self.y, self.plan, self.out, weights=self.weights, residual=self.shared)
        B.expert_combine_backward(self.dout, self.plan, y=self.y, weights=self.weights, dy=self.dy, dweights=self.dweights)
        B.expert_linear_backward(self.a1, self.w2, self.plan, self.dy, dx=self.da, dweight=self.dw2, workspace=self.ws, status=st)
        B.expert_linear_backward(self.x, self.w1, self.plan, self.da, dx=self.dz, dweight=self.dw1, preact=self.z1, activation="silu",
                                 gated=True, gather=True, workspace=self.ws, status=st)
        B.expert_combine(self.dz, self.plan, self.dx)
        B.route_experts_backward(logits, self.ids, self.dweights, self.dlogits, scoring="sigmoid")
        B.linear_backward(self.as_, self.s2, self.dout, dx=self.das, dweight=self.ds2, workspace=self.ws, status=st)
        B.linear_backward(self.x, self.s1, self.das, dweight=self.ds1, preact=self.zs, activation="silu", gated=True,
                          workspace=self.ws, status=st)

    def results(self):
        return [self.out, self.weights, self.dw1, self.dw2, self.ds1, self.ds2, self.dx, self.dlogits]

    def reference(self):
        """The same by autograd in 64 bits, the choice of experts taken from the block."""
        f = lambda v: v.double().requires_grad_(True)
        x, w1, w2, s1, s2 = f(self.x), f(self.w1), f(self.w2), f(self.s1), f(self.s2)
        logits = (self.x.double() @ self.router[0].double().T).requires_grad_(True)
        ids = self.ids.long()
        gate = lambda z: act64(z[:, : self.h], "silu") * z[:, self.h:]
        w = torch.sigmoid(logits).gather(1, ids)
        w = w / w.sum(1, keepdim=True)
        parts = []
        for e in range(self.e):
            y = gate(x @ w1[e].T) @ w2[e].T
            parts.append(y * (w * (ids == e)).sum(1, keepdim=True))
        routed = sum(parts)
        # the block's dx is that of the routed part alone
        dx, = torch.autograd.grad((routed * self.dout.double()).sum(), x, retain_graph=True)
        out = self.x.double() + gate(self.x.double() @ s1.T) @ s2.T + routed
        g = torch.autograd.grad((out * self.dout.double()).sum(), [w1, w2, s1, s2, logits])
        return [v.detach() for v in (out, w)] + [g[0], g[1], g[2], g[3], dx, g[4]]

    def check(self):
        self.B.check_status(self.status)
        # a chain of four to five stores of 2^-8 each, relative to a result's own size (rms), eight times over
        for got, want in zip(self.results(), self.reference()):
            rms = float(want.square().mean().sqrt())
            assert float((got.double() - want).abs().max()) <= 8 * 5 * 2.0 ** -8 * max(rms, float(want.abs().max()) / 8)
            assert float((got.double() - want).square().mean().sqrt()) <= 5 * 2.0 ** -8 * rms


def test_block(B):
    block = Block(B)
    block.run()
    block.check()


def test_block_long(B):
    block = Block(B, t=1500, k=4, e=16, d=512, h=264, seed=20)
    block.run()
    block.check()


def test_block_captured_and_replayed(B):
    """One graph of the whole chain, replayed on new contents; a second graph of another block in between."""
    first, second = Block(B), Block(B, t=33, seed=40)
    want = []
    graphs = []
    for block in (first, second):
        block.run()  # set-up outside the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            block.run()
        graphs.append(graph)
    for seed in (60, 61):
        first.x.copy_(rand(seed, first.t, first.d))
        second.x.copy_(rand(seed + 5, second.t, second.d))
        for v in first.results() + second.results():
            v.zero_()
        graphs[0].replay()
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        first.check()
        second.check()
        kept = [v.clone() for v in first.results()]
        first.run()
        assert all(torch.equal(a, b) for a, b in zip(kept, first.results()))  # eager gives the same bits


def test_block_on_another_stream(B):
    """Two blocks at once on streams of their own, each behind work of its stream."""
    blocks = [Block(B, seed=80), Block(B, t=64, k=3, seed=90)]
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for _ in range(3):
        for block, stream in zip(blocks, streams):
            with torch.cuda.stream(stream):
                x = block.x.clone()
                block.x.fill_(float("nan"))
                torch.cuda._sleep(200000)
                block.x.copy_(x)
                block.run()
    torch.cuda.synchronize()
    for block in blocks:
        block.check()


def test_graph_with_branches(B):
    """Two products on forked streams, a copy and a third product behind the join, captured and replayed."""
    x, w = rand(1, 40, 256), [rand(i, 256, 256, scale=1 / 16) for i in (2, 3, 4)]
    new = lambda: torch.zeros(40, 256, device="cuda", dtype=torch.bfloat16)
    a, b, c, out = new(), new(), new(), new()
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        B.linear(x, w[0], a, activation="silu")
        with torch.cuda.stream(side):
            B.linear(x, w[1], b, activation="relu")
        main.wait_stream(side)
        c.copy_(a)
        c.add_(b)
        B.linear(c, w[2], out, residual=b)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in (7, 8):
        x.copy_(rand(seed, 40, 256))
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (a, b, out)]
        for t in (a, b, c, out):
            t.fill_(float("nan"))
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(g, t) for g, t in zip(got, (a, b, out)))
        want, tol, _, _ = forward64(c, w[2], None, b, "none", False)
        bounded(out, want, tol + store(want, torch.bfloat16), "out")


def test_streams_are_named(B):
    """The ``stream`` argument: the call runs behind that stream's work, not the current one's."""
    x, w = rand(1, 64, 128), rand(2, 96, 128, scale=0.1)
    want = torch.empty(64, 96, device="cuda", dtype=torch.bfloat16)
    B.linear(x, w, want)
    out, side = torch.empty_like(want), torch.cuda.Stream()
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(500000)
        late.copy_(x)
    B.linear(late, w, out, stream=side)
    side.synchronize()
    assert torch.equal(out, want)


# ---------------------------------------------------------------- the same through tasks and modules
def test_linear_task(B):
    from flextensor_b200.runtime import build
    from flextensor_b200.scheduler import schedule_with_config
    from flextensor_b200.utils import Config
    key = "linear_linear_(64, 4096, 4096, 'gelu', False)_cuda(0)"
    x, w, b, r = rand(1, 64, 4096), rand(2, 4096, 4096, scale=1 / 64), rand(3, 4096), rand(4, 64, 4096)
    want, tol, _, _ = forward64(x, w, b, r, "gelu", False)
    for config in ({}, {"spatial": [[32], [1]], "reduce": [[2], [4]]}, {"spatial": [[128], [2]], "reduce": [[0], [0]]}):
        s, bufs = schedule_with_config(key, Config([config], None))
        func = build(s, bufs, "cuda")
        out = torch.full((64, 4096), float("nan"), device="cuda", dtype=torch.bfloat16)
        func(x, w, b, r, out)
        func.check()
        bounded(out, want, tol + store(want, torch.bfloat16), str(config))
    assert func.time_evaluator(func.entry_name, None, number=3)(x, w, b, r, out).mean < 1e-2


def test_linear_search(B):
    from flextensor_b200 import scheduler as S
    from flextensor_b200.measure import InProcessMeasurer
    import numpy as np
    S.VERBOSE = False
    np.random.seed(0)
    torch.manual_seed(0)
    key = "linear_linear_(64, 4096, 4096, 'gelu', False)_cuda(0)"
    plan, bufs, configs = S.schedule(key, op_trial=3, op_stop=2, timeout=10, parallel=1, number=3, measurer=InProcessMeasurer(0))
    x, w, b, r = rand(1, 64, 4096), rand(2, 4096, 4096, scale=1 / 64), rand(3, 4096), rand(4, 64, 4096)
    out = torch.empty(64, 4096, device="cuda", dtype=torch.bfloat16)
    plan.build()(x, w, b, r, out)
    want, tol, _, _ = forward64(x, w, b, r, "gelu", False)
    bounded(out, want, tol + store(want, torch.bfloat16), "found")


def test_expert_ffn_task_captured(B):
    from flextensor_b200.runtime import build
    from flextensor_b200.scheduler import schedule_with_config
    from flextensor_b200.utils import Config
    t, e, k, d, h = 8, 64, 8, 2048, 1024
    s, bufs = schedule_with_config("experts_expert_ffn_(8, 64, 8, 2048, 1024)_cuda(0)", Config([], None))
    func = build(s, bufs, "cuda")
    from flextensor_b200.runtime import torch_dtype
    arrays = [torch.zeros(tuple(int(v) for v in b.shape), device="cuda", dtype=torch_dtype(b.dtype)) for b in bufs]
    x, logits, w1, w2 = arrays[:4]
    w1.copy_(rand(3, e, 2 * h, d, scale=d ** -0.5))
    w2.copy_(rand(4, e, d, h, scale=h ** -0.5))
    call = func.capture(*arrays)
    for seed in (10, 20):
        x.copy_(rand(seed, t, d))
        logits.copy_(rand(seed + 1, t, e, dtype=torch.float32))
        call.replay()
        torch.cuda.synchronize()
        func.check()
        ids, weights = route64(logits, k, None, "softmax", 1, 1, True, 1.0)
        assert torch.equal(arrays[4], ids)
        want = x.double()
        for i in range(e):
            mine = weights * (ids == i)
            rows = mine.sum(1) > 0
            if rows.any():
                z = x[rows].double() @ w1[i].double().T
                want[rows] += mine[rows].sum(1, keepdim=True) * ((act64(z[:, :h], "silu") * z[:, h:]) @ w2[i].double().T)
        # three stores on the way (hidden, y, out), the first two scaled by weights of at most one
        assert float((arrays[-1].double() - want).abs().max()) <= 8 * 3 * 2.0 ** -8 * float(want.square().mean().sqrt() + 1)
