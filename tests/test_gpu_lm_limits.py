"""The feed-forward operators where their arithmetic is weakest: scores far below one, the tail of GELU, finite values whose
powers overflow, rows that a plan does not fill.  Definitions, bounds and helpers as in ``test_gpu_lm``."""
import math

import pytest
import torch

from test_gpu_lm import B, E, STEP, act64, bounded, dz64, rand, route64, scores64, slope64, status  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- scores far below one
def routed(B, logits, k, **settings):
    ids = torch.full((logits.shape[0], k), -7, device="cuda", dtype=torch.int32)
    weights = torch.full((logits.shape[0], k), float("nan"), device="cuda")
    B.route_experts(logits, ids, weights, **settings)
    return ids, weights


def test_route_groups_of_vanishing_scores(B):
    """sigmoid(-87.4) + sigmoid(-87.4) = 2.2e-38 against sigmoid(-87.3) + sigmoid(-95) = 1.2e-38."""
    logits = torch.tensor([[-87.4, -87.4, -87.3, -95.0], [-87.3, -95.0, -87.4, -87.4]], device="cuda")
    ids, weights = routed(B, logits, 2, scoring="sigmoid", groups=2, top_groups=1)
    assert ids.tolist() == [[0, 1], [2, 3]]
    assert torch.allclose(weights, torch.full((2, 2), 0.5, device="cuda"), atol=1e-6)


@pytest.mark.parametrize("e,groups", [(32, 2), (64, 2), (60, 3), (256, 4)])
@pytest.mark.parametrize("bias", [None, "zeros", "tiny"])
def test_route_group_sums_of_low_scores(B, e, groups, bias):
    """Rows of logits between -95 and -6 whose groups' sums differ by less than the error of a fast exponential there (it
    grows with the logit): each group has two logits a few fp32 steps from the other groups', and nothing else near."""
    t, size = 8192, e // groups
    gen = torch.Generator().manual_seed(e + groups)
    level = -6 - 89 * torch.rand(t, 1, generator=gen, dtype=torch.float64)
    step = 2.0 ** (torch.floor(torch.log2(-level)) - 23)
    logits = (level - 12).expand(t, e).reshape(t, groups, size).clone()
    first = torch.randint(-6, 7, (t, groups), generator=gen)
    second = torch.randint(-2, 3, (t, groups), generator=gen) - first
    logits[:, :, 1] = level + step * first
    logits[:, :, size - 1] = level - 0.25 + step * second
    logits = logits.reshape(t, e).float().cuda()
    b = None
    if bias is not None:
        b = torch.zeros(e, device="cuda")
        if bias == "tiny":  # one that moves nothing but the highest rows
            b[::3] = 2.0 ** -40
    ids, weights = routed(B, logits, 2, bias=b, scoring="sigmoid", groups=groups, top_groups=1)
    want_ids, want = route64(logits, 2, b, "sigmoid", groups, 1, True, 1.0)
    assert torch.equal(ids, want_ids), int((ids != want_ids).any(1).sum())
    bounded(weights, want, (32 + e / 8) * E * want.abs(), "weights")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_rows_over_a_wide_range(B, scoring, dtype, groups, top_groups):
    """Levels from -95 to 30 with spreads from a hundredth to ten: every regime of both scorings."""
    t, e, k = 1024, 64, 6
    gen = torch.Generator().manual_seed(11)
    level = 30 - 125 * torch.rand(t, 1, generator=gen)
    spread = 10.0 ** (1 - 3 * torch.rand(t, 1, generator=gen))
    logits = (level + spread * torch.randn(t, e, generator=gen)).to(dtype).cuda()
    ids, weights = routed(B, logits, k, scoring=scoring, groups=groups, top_groups=top_groups)
    want_ids, want = route64(logits, k, None, scoring, groups, top_groups, True, 1.0)
    assert torch.equal(ids, want_ids), int((ids != want_ids).any(1).sum())
    bounded(weights, want, (32 + e / 8) * E * want.abs() + 1e-37, "weights")


# ---------------------------------------------------------------- plans that the caller made
@pytest.mark.parametrize("width", [72, 20])
def test_places_without_a_row(B, status, width):
    """A place inside an expert's run whose order names no row (-1, or one past the tokens) is a row of zeros, forward and
    backward, whatever the workspace held."""
    t, k, e, n = 12, 2, 3, 40
    order = torch.arange(t * k, dtype=torch.int32)
    order[3], order[4], order[13] = -1, t * k, 2 ** 31 - 1
    offsets = torch.tensor([0, 9, 9, 20], dtype=torch.int32)
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    plan = B.ExpertPlan.over(t, k, e, offsets.cuda(), order.cuda(), slots.cuda())
    x, w, b = rand(1, t, width), rand(2, e, n, width, scale=0.2), rand(3, e, n)
    dy = rand(4, t * k, n)
    rows = torch.zeros(20, width, device="cuda", dtype=torch.float64)
    for place in range(20):
        if 0 <= int(order[place]) < t * k:
            rows[place] = x[int(order[place]) // k].double()
    out = torch.full((t * k, n), 7.0, device="cuda", dtype=torch.bfloat16)
    B.expert_linear(x, w, plan, out, bias=b, gather=True, status=status)
    dx, dw, db = torch.full((t * k, width), 7.0, device="cuda", dtype=torch.bfloat16), torch.empty_like(w), torch.empty_like(b)
    ws = torch.full((B.expert_linear_backward_workspace_bytes(plan, n, width),), 255, dtype=torch.uint8, device="cuda")  # NaN
    B.expert_linear_backward(x, w, plan, dy, dx=dx, dweight=dw, dbias=db, gather=True, workspace=ws, status=status)
    for i, (a, c) in enumerate(((0, 9), (9, 9), (9, 20))):
        z = rows[a:c] @ w[i].double().T + b[i].double()
        size = rows[a:c].abs() @ w[i].double().abs().T + b[i].double().abs()
        bounded(out[a:c], z, 2 * (width + 2) * E * size + STEP[torch.bfloat16] * z.abs(), "out %d" % i)
        g = dy[a:c].double()
        want = g.T @ rows[a:c]
        bounded(dw[i], want, 2 * 32 * E * (g.abs().T @ rows[a:c].abs()) + STEP[torch.bfloat16] * want.abs(), "dw %d" % i)
        bounded(db[i], g.sum(0), 100 * E * g.abs().sum(0) + STEP[torch.bfloat16] * g.sum(0).abs(), "db %d" % i)
    assert (out[20:] == 7).all() and (dx[20:] == 7).all()


# ---------------------------------------------------------------- GELU's tail
def tail(dtype):
    """z from -3 to -8 (fp16: to -5, where its results end), exact in the type."""
    z = -torch.linspace(3, 8 if dtype == torch.bfloat16 else 5, 512)
    return z.to(dtype).cuda()


def relative(got, want, dtype, what):
    """Half a step of the result's type, and 2^-16 of the value for the arithmetic: the exponent of the bell is z^2 / 2 with
    two roundings of 2^-24, 2^-18.2 of the value at z = -8, the fast exponential adds 2^-22 + |z^2 / 2| 2^-24 (2^-18.9) and
    the rest a few 2^-22.  fp16 has a smallest step of 2^-24."""
    bounded(got, want, (STEP[dtype] + 2.0 ** -16) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0), what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gated", [False, True])
def test_gelu_tail(B, status, dtype, gated):
    z = tail(dtype)
    n = z.numel()
    w = torch.zeros(n * (2 if gated else 1), 64, device="cuda", dtype=dtype)
    w[:n, 0] = z
    if gated:
        w[n:, 0] = 4.0
    x = torch.zeros(3, 64, device="cuda", dtype=dtype)
    x[:, 0] = 1
    for cfg in (None, {"tile_n": 16, "split_k": 1}, {"cluster": 2}):
        out = torch.empty(3, n, device="cuda", dtype=dtype)
        B.linear(x, w, out, activation="gelu", gated=gated, cfg=cfg, status=status)
        want = act64(z.double(), "gelu") * (4 if gated else 1)
        relative(out, want.expand(3, n), dtype, "gelu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_slope_in_the_tail(B, status, dtype):
    """The bias gradient of one token is act'(z) itself, rounded once."""
    z = tail(dtype)[None]
    n = z.shape[1]
    dy = torch.ones(1, n, device="cuda", dtype=dtype)
    db = torch.empty(n, device="cuda", dtype=dtype)
    ws = torch.empty(B.linear_backward_workspace_bytes(1, n, 64), dtype=torch.uint8, device="cuda")
    B.linear_backward(rand(1, 1, 64, dtype=dtype), rand(2, n, 64, dtype=dtype), dy, dbias=db, preact=z, activation="gelu",
                      workspace=ws, status=status)
    relative(db, slope64(z[0].double(), "gelu"), dtype, "slope")


# ---------------------------------------------------------------- finite values whose powers overflow
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True])
def test_huge_preactivations(B, status, act, gated):
    """z up to the type's largest: every activation is z or 0 there and its slope 1 or 0, without a NaN on the way."""
    huge = torch.tensor([1e4, 1e10, 2e13, 1e19, 2e19, 1e25, 1e30, 3e38] * 8).to(torch.bfloat16)
    z = torch.cat([huge, -huge])[None].cuda()
    n = z.shape[1]
    zz = torch.cat([z, torch.full_like(z, 0.5)], dim=1) if gated else z
    w = torch.zeros(zz.shape[1], 64, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = zz[0]
    x = torch.zeros(1, 64, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    out = torch.empty(1, n, device="cuda", dtype=torch.bfloat16)
    B.linear(x, w, out, activation=act, gated=gated, status=status)
    want = act64(z.double(), act) * (0.5 if gated else 1)
    bounded(out, want, STEP[torch.bfloat16] * want.abs(), act)
    dy, db = torch.ones_like(out), torch.empty(zz.shape[1], device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(B.linear_backward_workspace_bytes(1, n, 64, gated), dtype=torch.uint8, device="cuda")
    B.linear_backward(x, w, dy, dbias=db, preact=zz, activation=act, gated=gated, workspace=ws, status=status)
    want = dz64(dy, zz, act, gated)[0]
    bounded(db, want, STEP[torch.bfloat16] * want.abs(), act + " slope")


@pytest.mark.parametrize("level", [-12.0, -25.0, -45.0, -62.0, -68.0, -75.0])
@pytest.mark.parametrize("size", [1e-20, 1e-13, 1.0, 1e12])
def test_route_backward_of_low_scores(B, level, size):
    """Scaled sigmoid weights: their gradient is that of a softmax over the chosen logits however small the scores and the
    incoming gradients are; no product of the two may leave the range of fp32 on the way."""
    t, e, k = 40, 64, 6
    logits = rand(5, t, e, dtype=torch.float32) * 0.5 + level
    ids, _ = routed(B, logits, k, scoring="sigmoid")
    dweights = rand(6, t, k, dtype=torch.float32) * size
    got = torch.full_like(logits, float("nan"))
    B.route_experts_backward(logits, ids, dweights, got, scoring="sigmoid")
    x = logits.double().requires_grad_(True)
    w = torch.sigmoid(x).gather(1, ids.long())
    want = torch.autograd.grad((w / w.sum(1, keepdim=True) * dweights).sum(), x)[0]
    # as in test_route_backward: a few steps of the row's largest term, which may cancel
    bounded(got, want, (64 + e / 4) * E * dweights.double().abs().amax(1, keepdim=True), "dlogits")


# ---------------------------------------------------------------- rows that a mask leaves little of
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_masked_rows_against_the_definition(B, scoring, dtype, groups, top_groups):
    t, e, k = 9, 40, 4
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
    logits[8, 10:] = -math.inf       # whole groups masked
    clean = torch.where(logits.isnan(), -math.inf, logits.double())
    for renorm in (True, False):
        ids, weights = routed(B, logits, k, scoring=scoring, groups=groups, top_groups=top_groups, renormalize=renorm)
        want_ids, want = route64(logits, k, None, scoring, groups, top_groups, renorm, 1.0)
        if scoring == "sigmoid" and renorm:
            # the ratios of the chosen scores where 64 bits lose the scores themselves: a softmax of log(sigmoid)
            part = torch.nn.functional.logsigmoid(clean.gather(1, ids.long()))
            want = torch.where(part.amax(1, keepdim=True) == -math.inf, 0.0, torch.softmax(part, 1).nan_to_num(0.0))
        if scoring == "softmax":
            # an infinite logit takes all of the mass (64 bits: inf - inf)
            want_ids[5, 0] = 7
            p5 = torch.zeros(e, dtype=torch.float64, device="cuda")
            p5[7] = 1
            want[5] = p5[ids[5].long()]
        assert torch.equal(ids[[r for r in range(t) if r != 5]], want_ids[[r for r in range(t) if r != 5]])
        assert ids[5, 0] == 7
        assert set(ids[4].tolist()) <= set(range(10 if groups > 1 else 5))
        bounded(weights, want, (32 + e / 8) * E * want.abs() + 1e-37, "weights")
        # gradients: rows with a finite largest logit, by the same definition in 64 bits
        dweights = rand(3, t, k, dtype=torch.float32)
        back = torch.full_like(logits, float("nan"))
        B.route_experts_backward(logits, ids, dweights, back, scoring=scoring, renormalize=renorm)
        assert torch.isfinite(back.float()).all()
        assert not back[1].any() and not back[6].any()
        rows = [0, 2, 3, 4, 7, 8]
        s = scores64(clean[rows], scoring)
        chosen, g = s.gather(1, ids[rows].long()), dweights[rows].double()
        r = want[rows]
        want = torch.zeros(len(rows), e, dtype=torch.float64, device="cuda")
        if renorm:
            d = r * (g - (r * g).sum(1, keepdim=True))
            want.scatter_add_(1, ids[rows].long(), d * (1 - chosen) if scoring == "sigmoid" else d)
        elif scoring == "sigmoid":
            want.scatter_add_(1, ids[rows].long(), g * chosen * (1 - chosen))
        else:
            dp = torch.zeros_like(want).scatter_add_(1, ids[rows].long(), g)
            want = s * (dp - (dp * s).sum(1, keepdim=True))
        bounded(back[rows], want, (64 + e / 4) * E * g.abs().amax(1, keepdim=True) + (STEP[dtype] * want.abs() + 2.0 ** -25), "dlogits")


def test_expert_ffn_task_without_its_residual(B):
    """The routed part of the block alone, against its own size: a lost or misplaced expert shows."""
    from flextensor_b200.runtime import build, torch_dtype
    from flextensor_b200.scheduler import schedule_with_config
    from flextensor_b200.utils import Config
    t, e, k, d, h = 8, 64, 8, 2048, 1024
    s, bufs = schedule_with_config("experts_expert_ffn_(8, 64, 8, 2048, 1024)_cuda(0)", Config([], None))
    func = build(s, bufs, "cuda")
    arrays = [torch.zeros(tuple(int(v) for v in b.shape), device="cuda", dtype=torch_dtype(b.dtype)) for b in bufs]
    x, logits, w1, w2 = arrays[:4]
    w1.copy_(rand(3, e, 2 * h, d, scale=d ** -0.5))
    w2.copy_(rand(4, e, d, h, scale=h ** -0.5))
    x.copy_(rand(10, t, d))
    logits.copy_(rand(11, t, e, dtype=torch.float32))
    func(*arrays)
    func.check()
    ids, weights = route64(logits, k, None, "softmax", 1, 1, True, 1.0)
    assert torch.equal(arrays[4], ids)
    routed_part, size = torch.zeros(t, d, device="cuda", dtype=torch.float64), torch.zeros(t, d, device="cuda", dtype=torch.float64)
    for i in range(e):
        share = (weights * (ids == i)).sum(1, keepdim=True)
        if bool((share > 0).any()):
            z = x.double() @ w1[i].double().T
            hidden = act64(z[:, :h], "silu") * z[:, h:]
            y = hidden @ w2[i].double().T
            # the hidden row and y are stored in bf16 on the way: 2^-8 of each; the first error passes w2, whose terms
            # have independent signs: eight standard deviations
            off = 8 * 2.0 ** -8 * (hidden.square() @ w2[i].double().square().T).sqrt()
            routed_part += share * y
            size += share * (2.0 ** -8 * y.abs() + off + 2.0 ** -18 * (hidden.abs() @ w2[i].double().abs().T))
    got = arrays[-1].double() - x.double()
    bounded(got, routed_part, size + 2.0 ** -8 * (routed_part + x.double()).abs(), "routed part")


# ---------------------------------------------------------------- tensors of more than 2^31 elements
def test_expert_weights_past_32_bits(B, status):
    """2.2e9 weights and as many of their gradient: the last expert's lie behind 2^31 of them."""
    t, k, e, n, width = 40, 2, 33, 8200, 8192
    ids = torch.stack([torch.arange(t) % e, torch.full((t,), e - 1)], dim=1).to(torch.int32)
    ids[:, 0] = torch.where(ids[:, 0] == e - 1, 0, ids[:, 0])
    plan = B.ExpertPlan(t, k, e)
    B.expert_plan(ids.cuda(), plan)
    x = rand(1, t, width)
    w = torch.empty(e, n, width, device="cuda", dtype=torch.bfloat16)
    for i in range(e):
        w[i].normal_(0, width ** -0.5, generator=torch.Generator(device="cuda").manual_seed(i))
    out, dy = torch.empty(t * k, n, device="cuda", dtype=torch.bfloat16), rand(2, t * k, n)
    B.expert_linear(x, w, plan, out, gather=True, status=status)
    dx, dw = torch.empty(t * k, width, device="cuda", dtype=torch.bfloat16), torch.empty_like(w)
    ws = torch.empty(B.expert_linear_backward_workspace_bytes(plan, n, width), dtype=torch.uint8, device="cuda")
    B.expert_linear_backward(x, w, plan, dy, dx=dx, dweight=dw, gather=True, workspace=ws, status=status)
    half = STEP[torch.bfloat16]
    for i in (0, e - 2, e - 1):
        a, c = plan.offsets[i:i + 2].tolist()
        rows, g, wi = x[plan.order[a:c].long() // k].double(), dy[a:c].double(), w[i].double()
        z = rows @ wi.T
        bounded(out[a:c], z, 2 * (width + 2) * E * (rows.abs() @ wi.abs().T) + half * z.abs(), "out")
        want = g @ wi
        bounded(dx[a:c], want, 2 * (n + 2) * E * (g.abs() @ wi.abs()) + half * want.abs(), "dx")
        want = g.T @ rows
        bounded(dw[i], want, 2 * (c - a + 2) * E * (g.abs().T @ rows.abs()) + half * want.abs(), "dw")


def test_sorted_rows_past_32_bits(B, status):
    """2.2e9 elements of y in the weighted sum and its gradient, and of x by place in a weight gradient."""
    t, k, n = 41000, 2, 27000
    plan = B.ExpertPlan(t, k, 2)
    ids = torch.tensor([[0, 1]], dtype=torch.int32).repeat(t, 1).cuda()
    B.expert_plan(ids, plan)
    y = torch.empty(t * k, n, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    weights, out = torch.rand(t, k, device="cuda"), torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    B.expert_combine(y, plan, out, weights=weights)
    dy, dweights = torch.empty_like(y), torch.empty_like(weights)
    B.expert_combine_backward(out, plan, y=y, weights=weights, dy=dy, dweights=dweights)
    half = STEP[torch.bfloat16]
    for i in (0, 20000, 39600, t - 1):
        part = torch.stack([y[i], y[t + i]]).double()
        terms = part * weights[i].double()[:, None]
        bounded(out[i], terms.sum(0), 6 * E * terms.abs().sum(0) + half * terms.sum(0).abs(), "out")
        want = out[i].double() * weights[i].double()[:, None]
        bounded(torch.stack([dy[i], dy[t + i]]), want, E * want.abs() + half * want.abs(), "dy")
        dots = part * out[i].double()
        bounded(dweights[i], dots.sum(1), 2 * (n + 2) * E * dots.abs().sum(1), "dweights")
    del y, dy, out
    t, k, n, width = 33800, 8, 8, 8192
    plan = B.ExpertPlan(t, k, 2)
    ids = torch.arange(8, dtype=torch.int32).remainder(2).repeat(t, 1).cuda()
    B.expert_plan(ids, plan)
    x, w, dy = rand(3, t, width), rand(4, 2, n, width), rand(5, t * k, n)
    dw = torch.empty_like(w)
    ws = torch.empty(B.expert_linear_backward_workspace_bytes(plan, n, width), dtype=torch.uint8, device="cuda")
    B.expert_linear_backward(x, w, plan, dy, dweight=dw, gather=True, workspace=ws, status=status)
    for i in range(2):
        a, c = plan.offsets[i:i + 2].tolist()
        token = plan.order[a:c].long() // k
        g = torch.zeros(t, n, dtype=torch.float64, device="cuda").index_add_(0, token, dy[a:c].double())
        size = torch.zeros(t, n, dtype=torch.float64, device="cuda").index_add_(0, token, dy[a:c].double().abs())
        want = g.T @ x.double()
        # sums of 135200 terms: the bound of a sum one after the other is far above what is lost; their size, not it, shows
        # a wrong row
        bounded(dw[i], want, 2.0 ** -14 * (size.T @ x.double().abs()) + half * want.abs(), "dw")


def test_logits_past_32_bits(B):
    """2.15e9 logits: the last tokens' lie behind 2^31 of them."""
    t, e, k = 2100000, 1024, 4
    logits = torch.empty(t, e, device="cuda", dtype=torch.bfloat16)
    logits[:-64] = -1.0
    logits[-64:] = rand(1, 64, e)
    logits[:64] = rand(2, 64, e)
    ids, weights = routed(B, logits, k)
    dweights, back = torch.ones_like(weights), torch.full_like(logits, float("nan"))
    dweights[:, 0] = 2.0
    B.route_experts_backward(logits, ids, dweights, back)
    for rows in (slice(0, 64), slice(t - 64, t)):
        want_ids, want = route64(logits[rows], k, None, "softmax", 1, 1, True, 1.0)
        assert torch.equal(ids[rows], want_ids)
        bounded(weights[rows], want, (32 + e / 8) * E * want.abs(), "weights")
        g = want * (dweights[rows].double() - (want * dweights[rows].double()).sum(1, keepdim=True))
        full = torch.zeros(64, e, dtype=torch.float64, device="cuda").scatter_(1, want_ids.long(), g)
        bounded(back[rows], full, 320 * E * 2 + STEP[torch.bfloat16] * full.abs(), "dlogits")
    assert ids[1000000].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True])
def test_slopes_at_zero(B, status, act, gated):
    """z of 0 and -0: relu's slope is 0 there, as the entry says, GELU's and SiLU's one half."""
    n, k = 16, 64
    z = torch.tensor([0.0, -0.0] * 8, dtype=torch.bfloat16)[None]
    zz = torch.cat([z, torch.full_like(z, 3.0)], dim=1).cuda() if gated else z.cuda()
    dy, db = torch.full((1, n), 2.0, device="cuda", dtype=torch.bfloat16), torch.empty(zz.shape[1], device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(B.linear_backward_workspace_bytes(1, n, k, gated), dtype=torch.uint8, device="cuda")
    w = rand(2, zz.shape[1], k)
    B.linear_backward(rand(1, 1, k), w, dy, dbias=db, preact=zz, activation=act, gated=gated, workspace=ws, status=status)
    slope = {"none": 1.0, "relu": 0.0}.get(act, 0.5)
    assert (db[:n] == 2 * slope * (3 if gated else 1)).all() and not db[n:].any()
