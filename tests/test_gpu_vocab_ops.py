"""GPU: the 4-bit LM head, the embedding lookup and its gradient, token
log-probabilities and the policy loss, against their 64-bit definitions with
tolerances counted from the roundings (tests/vocab_ref.py)."""
import math

import pytest
import torch

from tests import vocab_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def near(got, ref, tol):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - ref).abs() / tol)[bad].max()),
                                 bad.nonzero()[:3].tolist())


def w4_inputs(V, d, g, stype, zeros, seed):
    G = gen(seed)
    codes = torch.randint(0, 256, (V, d // 2), device="cuda", dtype=torch.uint8, generator=G)
    scales = ((torch.rand(V, d // g, device="cuda", generator=G) + 0.3) / math.sqrt(d)).to(stype)
    z = torch.randint(0, 16, (V, d // g), device="cuda", dtype=torch.uint8, generator=G) if zeros else None
    return codes, scales, z


W4_CASES = [
    # B, V, d, group, scale type, zero points, output type
    (1, 1, 32, 32, F32, False, F32),             # the smallest call
    (1, 1000, 256, 128, BF16, False, F32),
    (2, 257, 128, 128, BF16, True, BF16),        # one row past a tile; one block
    (16, 4099, 1024, 32, F32, True, F32),        # codec head, fine groups
    (17, 2049, 96, 32, BF16, False, BF16),       # d inside one block
    (33, 1500, 416, 32, F32, True, F32),         # d = 3 blocks and a group
    (48, 777, 1600, 64, BF16, False, F32),       # columns beyond the MMA's N
    (64, 20000, 2048, 128, BF16, True, BF16),
    (65, 515, 192, 64, F32, False, F32),         # last stage of one block
    (100, 3001, 4096, 64, BF16, True, F32),
    (128, 5000, 640, 128, F32, False, BF16),
    (129, 1111, 512, 32, BF16, True, F32),       # two chunks of rows
    (200, 2500, 1024, 64, BF16, False, BF16),
    (256, 900, 2048, 128, F32, True, F32),
]


@pytest.mark.parametrize("B,V,d,g,stype,zeros,odt", W4_CASES)
def test_lmhead_w4(B, V, d, g, stype, zeros, odt):
    from mstar_rs_b200 import kernel

    codes, scales, z = w4_inputs(V, d, g, stype, zeros, B + V + d)
    hidden = torch.randn(B, d, device="cuda", generator=gen(d)).to(BF16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = kernel.lmhead_logits_w4(hidden, codes, scales, zeros=z, dtype=odt, status=status)
    again = kernel.lmhead_logits_w4(hidden, codes, scales, zeros=z, dtype=odt, status=status)
    ref, tol = R.head(hidden, codes, scales, z, odt, parts=16)
    near(out, ref, tol + 1e-30)
    assert torch.equal(out, again)
    assert status.item() == 0


def test_lmhead_w4_strided_rows():
    """Hidden rows with a stride and an odd start, logits inside a wider
    buffer: only [:, :V] is written."""
    from mstar_rs_b200 import kernel

    B, V, d = 5, 1001, 256
    codes, scales, z = w4_inputs(V, d, 64, BF16, True, 3)
    wide = torch.randn(B, d + 33, device="cuda", generator=gen(1)).to(BF16)
    hidden = wide[:, 3:3 + d]
    buf = torch.full((B, V + 23), 7.0, device="cuda")
    kernel.lmhead_logits_w4(hidden, codes, scales, zeros=z, out=buf[:, 1:1 + V])
    ref, tol = R.head(hidden, codes, scales, z, F32, parts=16)
    near(buf[:, 1:1 + V], ref, tol)
    assert bool((buf[:, :1] == 7).all()) and bool((buf[:, 1 + V:] == 7).all())


def test_lmhead_w4_zero_scales_and_extremes():
    """Zero scales give zeros; every code at its zero point too; large hidden
    values pass through exactly."""
    from mstar_rs_b200 import kernel

    V, d = 300, 128
    codes = torch.full((V, d // 2), 0x88, device="cuda", dtype=torch.uint8)
    codes[1] = 0x0F  # even columns 15, odd 0
    scales = torch.ones(V, 1, device="cuda")
    scales[2] = 0.0
    codes[2] = 0xFF
    hidden = torch.full((2, d), 2.0 ** 100, device="cuda").to(BF16)
    hidden[1] = -(2.0 ** -100)
    out = kernel.lmhead_logits_w4(hidden, codes, scales)
    want = torch.zeros(2, V, device="cuda")
    want[0, 1], want[1, 1] = (7 - 8) * 64 * 2.0 ** 100, -(7 - 8) * 64 * 2.0 ** -100
    assert torch.equal(out, want)


@pytest.mark.parametrize("B,V,d,dtype", [(64, 151936, 2048, "bf16"), (1, 156940, 1024, "f32"), (24, 32000, 512, "bf16"),
                                         (130, 4096, 256, "f32")])
def test_lmhead_step_w4_matches_the_two_calls(B, V, d, dtype):
    from mstar_rs_b200 import kernel
    from mstar_rs_b200 import workloads as W

    case = W.qwen_mixed(seed=5, B=B, V=V)
    case.dtype = dtype
    kw = W.to_device(case)
    kw.pop("logits")
    codes, scales, z = w4_inputs(V, d, 128, BF16, True, 9)
    hidden = torch.randn(B, d, device="cuda", generator=gen(4)).to(BF16)
    tdt = BF16 if dtype == "bf16" else F32
    logits = torch.empty(B, V, dtype=tdt, device="cuda")
    ids, ids2 = (torch.zeros(B, dtype=torch.int64, device="cuda") for _ in range(2))
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    kernel.lmhead_step_w4(hidden, codes, scales, logits, zeros=z, status=st, **kw, out_ids=ids)
    ref = kernel.lmhead_logits_w4(hidden, codes, scales, zeros=z, dtype=tdt)
    kernel.sampler_step(ref, **kw, out_ids=ids2)
    assert torch.equal(logits, ref) and torch.equal(ids, ids2)
    assert st.item() == 0


# ------------------------------------------------------------ lookup


@pytest.mark.parametrize("shape,V,d,tt,ot", [
    ((1,), 1, 1, F32, F32), ((64,), 1000, 2048, BF16, BF16), ((3, 7), 100, 501, BF16, F32),
    ((1000,), 333, 96, F32, BF16), ((5,), 50, 34, BF16, BF16), ((77,), 4099, 1023, F32, F32),
    ((0,), 10, 8, BF16, BF16), ((2, 0, 3), 10, 8, F32, F32)])
def test_embed(shape, V, d, tt, ot):
    from mstar_rs_b200 import kernel

    table = torch.randn(V, d, device="cuda", generator=gen(d)).to(tt)
    ids = torch.randint(-2, V, shape, device="cuda", generator=gen(V))
    out = kernel.embed_tokens(ids, table, scale=math.sqrt(d), dtype=ot)
    assert out.shape == (*shape, d) and out.dtype == ot
    ref = torch.where((ids < 0)[..., None], 0.0, table.double()[ids.clamp(min=0)] * math.sqrt(d))
    near(out, ref, ref.abs() * (R.HALF[ot] + 2.0 ** -23))  # sqrt(d) as a float, the product, the rounding


def test_embed_strided_table_and_bad_ids():
    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel

    wide = torch.randn(50, 75, device="cuda", generator=gen(2)).to(BF16)
    table = wide[:, 3:67]  # 64 columns, odd start and stride
    ids = torch.tensor([0, 49, 50, -1, 2 ** 40, -2 ** 62, 7], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = kernel.embed_tokens(ids, table, status=status)
    want = torch.zeros(7, 64, device="cuda", dtype=BF16)
    want[[0, 1, 6]] = table[[0, 49, 7]]
    assert torch.equal(out, want)
    assert status.item() == N.STATUS_BAD_ID
    status.zero_()
    kernel.embed_tokens(ids[[0, 1, 3]].contiguous(), table, status=status)
    assert status.item() == 0  # padding is no error


@pytest.mark.parametrize("N_,V,d,g,st,z,ot", [(1, 1, 32, 32, F32, False, F32), (64, 999, 2048, 128, BF16, True, BF16),
                                              (333, 77, 192, 64, BF16, False, F32), (9, 5, 416, 32, F32, True, BF16)])
def test_embed_w4(N_, V, d, g, st, z, ot):
    from mstar_rs_b200 import kernel

    codes, scales, zeros = w4_inputs(V, d, g, st, z, N_)
    ids = torch.randint(-1, V + 1, (N_,), device="cuda", generator=gen(5))
    out = kernel.embed_tokens_w4(ids, codes, scales, zeros=zeros, scale=1.7, dtype=ot)
    ok = (ids >= 0) & (ids < V)
    ref = torch.where(ok[:, None], R.dequant(codes, scales, zeros)[ids.clamp(0, V - 1)] * 1.7, 0.0)
    near(out, ref, ref.abs() * (R.HALF[ot] + 3 * 2.0 ** -24))


GRAD_CASES = [
    # N, V, d, type, output type, ids
    (1, 1, 1, F32, F32, "all"), (5, 7, 3, BF16, BF16, "all"), (1000, 50, 64, BF16, F32, "all"),
    (3000, 151936, 128, BF16, BF16, "zipf"), (4097, 3, 130, F32, F32, "all"),        # runs over many chunks
    (2048, 5000, 2048, BF16, BF16, "one"),                                           # every token the same id
    (2049, 1200, 501, BF16, F32, "zipf"), (777, 300, 1026, F32, BF16, "ends"), (100, 40, 256, BF16, F32, "none"),
    (20000, 200000, 24, F32, F32, "zipf"),                                           # more ranges than SMs
]


@pytest.mark.parametrize("base", ["none", "apart", "in place"])
@pytest.mark.parametrize("N_,V,d,tt,ot,kind", GRAD_CASES)
def test_embed_grad(N_, V, d, tt, ot, kind, base):
    from mstar_rs_b200 import kernel

    G = gen(N_ + V)
    if kind == "all":
        ids = torch.randint(-1, V, (N_,), device="cuda", generator=G)
    elif kind == "zipf":
        u = torch.rand(N_, device="cuda", generator=G, dtype=torch.float64)
        ids = (torch.exp(u * math.log(V + 1)).long() - 1).clamp(0, V - 1)
    elif kind == "one":
        ids = torch.full((N_,), V - 1, device="cuda")
    elif kind == "ends":
        ids = torch.where(torch.rand(N_, device="cuda", generator=G) < 0.5, 0, V - 1)
    else:
        ids = torch.full((N_,), -1, device="cuda")
    dout = torch.randn(N_, d, device="cuda", generator=G).to(tt)
    b = None if base == "none" else torch.randn(V, d, device="cuda", generator=G).to(ot)
    ref, tol = R.embed_grad(ids, dout, V, 0.37, b, ot)
    tol = tol + ref.abs() * 2.0 ** -23  # 0.37 as a float
    keep = None if b is None else b.clone()
    out = kernel.embed_tokens_grad(ids, dout, V, scale=0.37, base=b, out=b if base == "in place" else None, dtype=ot)
    assert out.dtype == ot and out.shape == (V, d)
    near(out, ref, tol)
    if base == "apart":
        assert torch.equal(b, keep)
    if base != "in place":
        assert torch.equal(out, kernel.embed_tokens_grad(ids, dout, V, scale=0.37, base=b, dtype=ot))


def test_embed_grad_by_differences():
    """The lookup is linear, so its gradient applied to a change of the table
    is the change of sum(dout * lookup), up to the sums' roundings."""
    from mstar_rs_b200 import kernel

    V, d, n = 40, 24, 300
    G = gen(8)
    ids = torch.randint(-1, V, (n,), device="cuda", generator=G)
    dout = torch.randn(n, d, device="cuda", generator=G)
    step = torch.randn(V, d, device="cuda", generator=G)
    grad = kernel.embed_tokens_grad(ids, dout, V, scale=3.0)
    moved = kernel.embed_tokens(ids, step, scale=3.0)
    a = (moved.double() * dout.double()).sum()
    b = (grad.double() * step.double()).sum()
    size = (moved.double().abs() * dout.double().abs()).sum()
    assert abs(a - b) <= size * (n + 3) * 2.0 ** -24


def test_embed_grad_strided_and_bad_ids():
    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel

    wide = torch.randn(200, 77, device="cuda", generator=gen(3)).to(BF16)
    dout = wide[:, 5:70]
    ids = torch.randint(0, 30, (200,), device="cuda", generator=gen(4))
    ids[::7], ids[3], ids[10] = -5, 30, 2 ** 33 + 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = kernel.embed_tokens_grad(ids, dout, 30, status=status, dtype=F32)
    ref, tol = R.embed_grad(ids, dout, 30, 1.0, None, F32)
    near(out, ref, tol)
    assert status.item() == N.STATUS_BAD_ID


# ------------------------------------------------------------ log-probabilities and the policy loss


def row_inputs(n, V, dtype, seed, masked=0.0):
    G = gen(seed)
    x = torch.randn(n, V, device="cuda", generator=G) * 3
    ids = torch.randint(0, V, (n,), device="cuda", generator=G)
    if masked:
        x.masked_fill_(torch.rand(n, V, device="cuda", generator=G) < masked, -math.inf)
        x[torch.arange(n), ids] = 1.0
    if n > 3:
        ids[1], ids[3] = -1, V  # padding, and a bad id
    return x.to(dtype), ids


ROW_CASES = [(1, 1, F32), (1, 2, BF16), (5, 7, BF16), (64, 1000, BF16), (3, 32001, F32), (7, 151936, BF16),
             (2, 257152, F32), (300, 4097, F32), (1000, 128, BF16), (2, 600001, BF16), (1, 1000000, F32)]


@pytest.mark.parametrize("T", [1.0, 0.37])
@pytest.mark.parametrize("n,V,dtype", ROW_CASES)
def test_token_logprobs_and_gradient(n, V, dtype, T):
    from mstar_rs_b200 import kernel

    x, ids = row_inputs(n, V, dtype, n + V, masked=0.3 if V > 100 else 0.0)
    logp, lse = kernel.token_logprobs(x, ids, temperature=T)
    valid, rl, rp = R.rows(x, ids, T)
    near(lse, rl, R.SUM + rl.abs() * 2.0 ** -23)
    near(logp, rp, torch.where(valid, R.SUM + rp.abs() * 2.0 ** -23, 0.0))
    dlogp = torch.randn(n, device="cuda", generator=gen(1))
    out = kernel.token_logprobs_grad(x, ids, lse, dlogp, temperature=T)
    # the given lse, rounded to 32 bits, is the definition's here
    ref, tol = R.grad(x, ids, T, lse.double(), dlogp.double(), dtype, rel=2.0 ** -20)
    near(out, ref, tol)
    same = kernel.token_logprobs_grad(x, ids, lse, dlogp, temperature=T, out=x)  # in place
    assert same is x and torch.equal(x, out)


@pytest.mark.parametrize("n,V,dtype", ROW_CASES)
@pytest.mark.parametrize("old,ref,T", [(True, True, 1.0), (True, False, 0.6), (False, True, 1.7)])
def test_policy_loss(n, V, dtype, old, ref, T):
    from mstar_rs_b200 import kernel

    x, ids = row_inputs(n, V, dtype, n * 3 + V, masked=0.3 if V > 100 else 0.0)
    G = gen(7)
    _, _, lp = R.rows(x, ids, T)
    noise = torch.randn(n, device="cuda", generator=G, dtype=torch.float64) * 0.2
    r = noise.exp()
    noise += 0.02 * (((r - 0.9).abs() < 5e-3) | ((r - 1.3).abs() < 5e-3))  # off the border, where the gradient jumps
    olp = (lp - noise).float() if old else None
    rlp = (lp + 0.5 * torch.randn(n, device="cuda", generator=G)).float() if ref else None
    adv = torch.randn(n, device="cuda", generator=G)
    w = torch.rand(n, device="cuda", generator=G)
    beta = 0.1 if ref else 0.0
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(ref_logp=rlp, weights=w, temperature=T, clip_low=0.1, clip_high=0.3, kl_coef=beta, status=status)
    loss, logp, dx = kernel.policy_loss(x, ids, olp, adv, **kw)
    rloss, ltol, rlp_, d, dtol, lse = R.policy(x, ids, olp, adv, T, 0.1, 0.3, beta, rlp, w)
    near(loss, rloss, ltol)
    near(logp, rlp_, torch.where(R.rows(x, ids, T)[0], R.SUM + rlp_.abs() * 2.0 ** -23, 0.0))
    gref, gtol = R.grad(x, ids, T, lse, d, dtype)
    near(dx, gref, gtol + (dtol / T)[:, None] * 2)
    assert status.item() == (0x80 if n > 3 else 0)
    loss2, logp2, none = kernel.policy_loss(x, ids, olp, adv, **kw, grad=False)
    assert none is None and torch.equal(loss2, loss) and torch.equal(logp2, logp)
    _, _, same = kernel.policy_loss(x, ids, olp, adv, **kw, dlogits=x)  # in place
    assert same is x and torch.equal(x, dx)


def test_policy_gradient_by_differences():
    """(loss(x + h u) - loss(x - h u)) / 2h along random directions, in f32
    logits, against the gradient: within the third-order term (h^2 |u|^3-ish,
    h = 1e-2 on unit directions: under 1e-3 of the gradient's size) and the
    loss's own rounding over 2h."""
    from mstar_rs_b200 import kernel

    n, V = 6, 50
    G = gen(11)
    x = torch.randn(n, V, device="cuda", generator=G)
    ids = torch.randint(0, V, (n,), device="cuda", generator=G)
    _, _, lp = R.rows(x, ids, 1.0)
    old, ref = (lp - 0.05).float(), (lp + 0.3).float()  # ratio 1.05: inside the clip on both sides of every step
    adv = torch.randn(n, device="cuda", generator=G)
    kw = dict(ref_logp=ref, kl_coef=0.2)
    _, _, dx = kernel.policy_loss(x, ids, old, adv, **kw)
    h = 1e-2
    for k in range(8):
        u = torch.randn(n, V, device="cuda", generator=gen(20 + k))
        u /= u.norm(dim=1, keepdim=True)
        up = kernel.policy_loss(x + h * u, ids, old, adv, **kw, grad=False)[0].double()
        dn = kernel.policy_loss(x - h * u, ids, old, adv, **kw, grad=False)[0].double()
        num, ana = (up - dn) / (2 * h), (dx.double() * u.double()).sum(1)
        size = adv.double().abs() * 1.05 + 0.2 * 2
        assert bool(((num - ana).abs() <= size * (2e-4 + 2 * 1.3e-5 / h)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5, 1000, 40000])
def test_rows_at_the_edges(V, dtype):
    """Nothing left of a row; a mask of the type's lowest value; a row of that
    value alone (uniform); huge values; a masked id; NaN and +inf."""
    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel

    low = torch.finfo(dtype).min
    x = torch.randn(9, V, device="cuda", generator=gen(V)).to(dtype)
    ids = torch.full((9,), 2, device="cuda")
    x[0] = -math.inf                       # empty
    x[1] = low                             # uniform at the lowest value
    x[2, 3:] = low                         # masked by it
    x[3, 1:] = -math.inf                   # one id left, and it is not the sampled one
    x[4, 2] = 3e38                         # all the weight on the id
    x[5, 4] = 3e38                         # none of it
    x[6, 0] = math.nan
    x[7, 0] = math.inf
    adv = torch.ones(9, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    logp, lse = kernel.token_logprobs(x, ids, status=status)
    assert status.item() == N.STATUS_EMPTY
    _, rl, rp = R.rows(x[:6], ids[:6], 1.0)
    assert logp[0] == -math.inf and lse[0] == -math.inf and logp[3] == -math.inf
    for i in (1, 2, 4, 5):
        assert abs(logp[i].double() - rp[i]) <= R.SUM + rp[i].abs() * 2.0 ** -23, i
    assert bool(torch.isnan(logp[6:8]).all()) and bool(torch.isfinite(logp[8]))
    for old in (None, torch.zeros(9, device="cuda")):
        loss, lp, dx = kernel.policy_loss(x, ids, old, adv, clip_high=1e30)
        assert torch.equal(lp.nan_to_num(1.0), logp.nan_to_num(1.0))
        assert loss[0] == 0 and bool((dx[0] == 0).all())           # empty: no loss, no gradient
        assert bool((dx[3] == 0).all())                            # a masked id: no gradient
        assert bool(torch.isfinite(loss[1:6]).all()) and bool(torch.isfinite(dx[:6].float()).all())
        assert bool(torch.isnan(loss[6:8]).all())
        r = torch.ones(()) if old is None else logp[1].exp().cpu()  # the uniform row: -r (onehot - 1/V)
        want = torch.full((V,), float(r) / V, dtype=torch.float64)
        want[2] -= float(r)
        near(dx[1].cpu(), want, want.abs() * (R.HALF[dtype] + 2e-5) + float(r) * 2.0 ** -22)
        assert bool((dx[2, 3:] == 0).all())
    g = kernel.token_logprobs_grad(x, ids, lse, adv)
    assert bool((g[0] == 0).all()) and bool((g[2, 3:] == 0).all()) and bool(torch.isfinite(g[8].float()).all())


def test_rows_strided_and_misaligned():
    """Rows inside a wider matrix, starting at an odd column, gradients into
    another layout: only the rows' own columns are written."""
    from mstar_rs_b200 import kernel

    n, V = 6, 999
    for dtype in (BF16, F32):
        for off in (1, 3, 5):
            wide = torch.randn(n, V + 31, device="cuda", generator=gen(off)).to(dtype)
            x = wide[:, off:off + V]
            ids = torch.randint(0, V, (n,), device="cuda", generator=gen(2))
            to = torch.full((n, V + 12), 5.0, device="cuda").to(dtype)
            adv = torch.randn(n, device="cuda", generator=gen(3))
            _, _, dx = kernel.policy_loss(x, ids, None, adv)
            _, _, dy = kernel.policy_loss(x, ids, None, adv, dlogits=to[:, 2:2 + V])
            assert torch.equal(dx, dy) and bool((to[:, :2] == 5).all()) and bool((to[:, 2 + V:] == 5).all())
            logp, lse = kernel.token_logprobs(x, ids)
            want = kernel.token_logprobs_grad(x.contiguous(), ids, lse, adv)
            got = kernel.token_logprobs_grad(x, ids, lse, adv, out=to[:, 1:1 + V])
            assert torch.equal(got, want)


# ------------------------------------------------------------ together, streams, graphs


def test_a_rollout_and_its_update():
    """The operators as they are used together: look up the sampled ids in
    the tied 4-bit table, project with it, sample, take the log-probabilities
    of what was sampled, then the policy loss on the same logits and the
    gradient of the lookup; captured once and replayed, each step equal to
    the eager calls'."""
    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel

    B, V, d = 12, 5003, 256
    w = torch.randn(V, d, device="cuda", generator=gen(1)) * 0.2
    codes, scales, zeros = kernel.quantize_w4(w, 64, zero_points=True)
    seed = torch.arange(B, dtype=torch.int64, device="cuda")

    def step(ids, offset, logits):
        x = kernel.embed_tokens_w4(ids, codes, scales, zeros=zeros, scale=math.sqrt(d))
        out = torch.empty_like(ids)
        kernel.lmhead_step_w4(x, codes, scales, logits, zeros=zeros, seed=seed, offset=offset, out_ids=out,
                              flags=N.FLAG_ADVANCE_OFFSET)
        logp, lse = kernel.token_logprobs(logits, out)
        loss, lp, dl = kernel.policy_loss(logits, out, logp, torch.ones_like(logp))
        dx = (dl @ w).to(BF16)
        dw = kernel.embed_tokens_grad(ids, dx, V, scale=math.sqrt(d), dtype=F32)
        return out, logp, loss, lp, dl, dw

    ids0 = torch.randint(0, V, (B,), device="cuda", generator=gen(2))
    off_e = torch.zeros(B, dtype=torch.int64, device="cuda")
    eager, ids = [], ids0
    for _ in range(3):
        r = step(ids, off_e, torch.empty(B, V, device="cuda"))
        eager.append([t.clone() for t in r])
        ids = r[0]
    assert bool((eager[0][1] == eager[0][3]).all())  # both take the same log-probabilities
    near(eager[0][2], torch.full((B,), -1.0, dtype=torch.float64, device="cuda"), 1e-6)  # ratio 1, advantage 1

    gids, goff, glog = ids0.clone(), torch.zeros_like(off_e), torch.empty(B, V, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step(gids, goff, glog)
    for want in eager:
        g.replay()
        for a, b in zip(res, want):
            assert torch.equal(a, b)
        gids.copy_(res[0])


def test_two_streams_at_once():
    """Calls on two streams, and two captured graphs replayed on two streams:
    each has its own scratch."""
    from mstar_rs_b200 import kernel

    V, d = 20000, 512
    codes, scales, _ = w4_inputs(V, d, 128, BF16, False, 5)
    hs = [torch.randn(b, d, device="cuda", generator=gen(b)).to(BF16) for b in (3, 40)]
    ids = [torch.randint(0, 900, (n,), device="cuda", generator=gen(n)) for n in (5000, 7000)]
    douts = [torch.randn(len(i), 96, device="cuda", generator=gen(9)).to(BF16) for i in ids]
    one = lambda k: (kernel.lmhead_logits_w4(hs[k], codes, scales), kernel.embed_tokens_grad(ids[k], douts[k], 900))  # noqa: E731
    want = [one(k) for k in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(one(k))
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, b) for r in got[k] for a, b in zip(r, want[k]))
    graphs = []
    for k in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = one(k)
        graphs.append((g, r))
    for _ in range(5):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(graphs[k][1], want[k]))


# ------------------------------------------------------------ refusals, sizes past 32 bits


def test_front_end_refusals():
    from mstar_rs_b200 import kernel as k

    dev = "cuda"
    x, ids, f = torch.zeros(4, 64, device=dev), torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(4, device=dev)
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8, device=dev), torch.ones(8, 1, device=dev)
    h = torch.zeros(4, 64, device=dev, dtype=BF16)
    cases = [
        (TypeError, lambda: k.token_logprobs(x.half(), ids)), (TypeError, lambda: k.token_logprobs(x, ids.int())),
        (ValueError, lambda: k.token_logprobs(x[0], ids)), (ValueError, lambda: k.token_logprobs(x, ids[:3])),
        (ValueError, lambda: k.token_logprobs(x.t(), ids)), (ValueError, lambda: k.token_logprobs(x, ids, temperature=0.0)),
        (ValueError, lambda: k.token_logprobs(x, ids.cpu())),
        (ValueError, lambda: k.token_logprobs(x[:1].expand(4, 64), ids)),  # rows on top of one another
        (ValueError, lambda: k.token_logprobs(x, ids, status=f)),
        (TypeError, lambda: k.token_logprobs_grad(x, ids, f, f.double())),
        (TypeError, lambda: k.token_logprobs_grad(x, ids, f, f, out=torch.zeros(4, 64, device=dev, dtype=BF16))),
        (ValueError, lambda: k.token_logprobs_grad(x[:, :60], ids, f, f, out=x[:, 4:])),  # overlapping, not the same
        (ValueError, lambda: k.policy_loss(x, ids, f, None)), (ValueError, lambda: k.policy_loss(x, ids, f, f, kl_coef=0.1)),
        (ValueError, lambda: k.policy_loss(x, ids, f, f, clip_low=2.0)),
        (ValueError, lambda: k.policy_loss(x, ids, f, f, kl_coef=math.nan, ref_logp=f)),
        (ValueError, lambda: k.policy_loss(x, ids, f, f, grad=False, dlogits=x)),
        (ValueError, lambda: k.policy_loss(x, ids, f[:2], f)),
        (TypeError, lambda: k.embed_tokens(ids, x.half())), (TypeError, lambda: k.embed_tokens(ids, x, dtype=torch.float16)),
        (ValueError, lambda: k.embed_tokens(ids, x, out=x)), (ValueError, lambda: k.embed_tokens(ids[::2], x)),
        (ValueError, lambda: k.embed_tokens(ids, x, out=torch.zeros(3, 64, device=dev))),
        (ValueError, lambda: k.embed_tokens_grad(ids, x[:3], 9)), (ValueError, lambda: k.embed_tokens_grad(ids, x, 0)),
        (ValueError, lambda: k.embed_tokens_grad(ids, x, 4, out=x)),
        (TypeError, lambda: k.embed_tokens_grad(ids, x, 4, base=torch.zeros(4, 64, device=dev), dtype=BF16)),
        (ValueError, lambda: k.embed_tokens_grad(ids, x, 9, base=torch.zeros(4, 64, device=dev))),
        (ValueError, lambda: k.embed_tokens_w4(ids, codes, scales, zeros=torch.zeros(8, 2, dtype=torch.uint8, device=dev))),
        (TypeError, lambda: k.embed_tokens_w4(ids, codes, scales.half())),
        (ValueError, lambda: k.embed_tokens_w4(ids, codes, torch.ones(8, 4, device=dev))),  # groups of 16
        (TypeError, lambda: k.lmhead_logits_w4(x, codes, scales)), (ValueError, lambda: k.lmhead_logits_w4(h[:, :32], codes, scales)),
        (ValueError, lambda: k.lmhead_logits_w4(torch.zeros(257, 64, device=dev, dtype=BF16), codes, scales)),
        (ValueError, lambda: k.lmhead_logits_w4(h, codes, scales, out=torch.zeros(4, 9, device=dev))),
        (ValueError, lambda: k.lmhead_logits_w4(h, codes, scales, workspace=f)),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
    assert bool((x == 0).all())


def test_nothing_to_do():
    """No rows: empty results, no launch; the lookup's gradient of no tokens
    is the base, or zeros."""
    from mstar_rs_b200 import kernel as k

    x, ids, f = torch.zeros(0, 64, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(0, device="cuda")
    assert k.token_logprobs(x, ids)[0].shape == (0,)
    assert k.token_logprobs_grad(x, ids, f, f).shape == (0, 64)
    assert k.policy_loss(x, ids, f, f)[2].shape == (0, 64)
    base = torch.randn(5, 64, device="cuda")
    assert bool((k.embed_tokens_grad(ids, x, 5) == 0).all())
    assert torch.equal(k.embed_tokens_grad(ids, x, 5, base=base), base)
    assert k.embed_tokens_grad(ids, x, 5, base=base, out=base) is base


def test_places_past_32_bits():
    """Rows, tables and weights whose last elements lie beyond 2^31 of them."""
    from mstar_rs_b200 import kernel as k

    V, n = 151936, 14300
    x = torch.zeros(n, V, device="cuda", dtype=BF16)
    x[-2:] = torch.randn(2, V, device="cuda", generator=gen(1)).to(BF16)
    ids = torch.full((n,), V - 1, device="cuda")
    adv = torch.ones(n, device="cuda")
    assert (n - 2) * V > 2 ** 31
    loss, logp, dx = k.policy_loss(x, ids, None, adv, dlogits=None)
    _, lse, lp = R.rows(x[-2:], ids[-2:], 1.0)
    near(logp[-2:], lp, R.SUM + lp.abs() * 2.0 ** -23)
    ref, tol = R.grad(x[-2:], ids[-2:], 1.0, lse, -adv[-2:].double(), BF16)
    near(dx[-2:], ref, tol)
    assert abs(float(logp[0]) + math.log(V)) <= R.SUM + 13 * 2.0 ** -23
    del x, dx, loss
    V, d = 1_700_000, 1300
    table = torch.zeros(V, d, device="cuda", dtype=BF16)
    table[-3:] = torch.randn(3, d, device="cuda", generator=gen(2)).to(BF16)
    ids = torch.tensor([V - 1, 0, V - 3], device="cuda")
    assert torch.equal(k.embed_tokens(ids, table), table[ids])
    del table
    dout = torch.randn(3, d, device="cuda", generator=gen(3)).to(BF16)
    g = k.embed_tokens_grad(ids, dout, V)
    assert torch.equal(g[ids], dout) and not bool(g[1:-3].any()) and not bool(g[-2].any())
    del g
    V, d = 1_100_000, 4096
    codes = torch.full((V, d // 2), 0x88, device="cuda", dtype=torch.uint8)
    codes[-5:] = torch.randint(0, 256, (5, d // 2), device="cuda", dtype=torch.uint8, generator=gen(4))
    scales = torch.full((V, d // 128), 0.01, device="cuda")
    hidden = torch.randn(2, d, device="cuda", generator=gen(5)).to(BF16)
    out = k.lmhead_logits_w4(hidden, codes, scales)
    ref, tol = R.head(hidden, codes[-5:], scales[-5:], None, F32, parts=16)
    near(out[:, -5:], ref, tol)
    assert not bool(out[:, :-5].any())
    assert torch.equal(k.embed_tokens_w4(torch.tensor([V - 2], device="cuda"), codes, scales, dtype=F32).double(),
                       R.dequant(codes[-2:-1], scales[-2:-1], None).float().double())


def test_another_stream_than_the_tensors_own():
    """Inputs made on one stream, the calls on another that waits for it."""
    from mstar_rs_b200 import kernel as k

    codes, scales, _ = w4_inputs(30000, 512, 64, BF16, False, 1)
    hidden = torch.randn(7, 512, device="cuda", generator=gen(2)).to(BF16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = k.lmhead_logits_w4(hidden, codes, scales)
        ids = out.argmax(1)
        logp, lse = k.token_logprobs(out, ids)
        g = k.embed_tokens_grad(ids, hidden, 30000, dtype=F32)
    torch.cuda.current_stream().wait_stream(s)
    ref, tol = R.head(hidden, codes, scales, None, F32, parts=16)
    near(out, ref, tol)
    _, _, lp = R.rows(out, ids, 1.0)
    near(logp, lp, R.SUM + lp.abs() * 2.0 ** -23)
    gref, gtol = R.embed_grad(ids, hidden, 30000, 1.0, None, F32)
    near(g, gref, gtol)


def test_infinities_and_nan_in_hidden_rows():
    """A row's infinity meets codes at their zero point as NaN and others as
    an infinity, as the products say; other rows keep theirs."""
    from mstar_rs_b200 import kernel as k

    V, d = 260, 256
    codes, scales, z = w4_inputs(V, d, 64, F32, True, 8)
    hidden = torch.randn(4, d, device="cuda", generator=gen(9)).to(BF16)
    hidden[1, 5], hidden[2, 7], hidden[3] = math.inf, math.nan, 0.0
    out = k.lmhead_logits_w4(hidden, codes, scales, zeros=z)
    want = hidden.double() @ R.dequant(codes, scales, z).t()
    assert torch.equal(out[1].isnan(), want[1].isnan()) and torch.equal(out[1] > 0, want[1] > 0)
    assert bool(out[1].isfinite().logical_not().all()) and bool(out[2].isnan().all()) and not bool(out[3].any())
    ref, tol = R.head(hidden[:1], codes, scales, z, F32, parts=16)
    near(out[:1], ref, tol)


def test_small_hidden_values_beside_a_large_one():
    """Values 2^-31 of the row's largest keep their bits; below that they are
    off by at most 2^-40 of it."""
    from mstar_rs_b200 import kernel as k

    V, d = 300, 128
    codes = torch.full((V, d // 2), 0x99, device="cuda", dtype=torch.uint8)  # every weight 1
    codes[:, 0] = 0x98  # column 0: weight 0
    scales = torch.ones(V, 1, device="cuda")
    for big in (1.0, 2.0 ** 100, 2.0 ** -90):
        for e in (20, 31, 36):
            hidden = torch.zeros(1, d, device="cuda")
            hidden[0, 0], hidden[0, 9] = big, big * 2.0 ** -e * 1.1015625
            hidden = hidden.to(BF16)
            out = k.lmhead_logits_w4(hidden, codes, scales)
            err = (out.double() - hidden[0, 9].double()).abs().max()
            assert err <= (0.0 if e <= 31 else big * 2.0 ** -40), (big, e, float(err))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_of_rows_far_from_zero(dtype):
    """Rows whose lse 32 bits cannot hold to log V: the softmax of the row
    itself, as the policy loss takes it.  An lse that is not the row's own (a
    part of a longer row) is taken as given."""
    from mstar_rs_b200 import kernel as k

    V = 3001
    low = torch.finfo(dtype).min
    for T in (1.0, 0.7, 1e-5):
        x = torch.randn(8, V, device="cuda", generator=gen(3)).to(dtype)
        x[0], x[1], x[2] = low, -1e10, 1e10
        x[3], x[3, 7] = -1e9, -math.inf
        x[4] = x[4] + 70000
        x[5], x[5, 1:] = 3e38, low
        x[6] = low
        x[6, :2] = -1e30
        ids = torch.tensor([5, 5, 0, 9, 5, 0, 1, 5], device="cuda")
        dlogp = torch.randn(8, device="cuda", generator=gen(4))
        logp, lse = k.token_logprobs(x, ids, temperature=T)
        got = k.token_logprobs_grad(x, ids, lse, dlogp, temperature=T)
        _, true, lp = R.rows(x, ids, T)
        near(logp, lp, R.SUM + lp.abs() * 2.0 ** -23)
        xd = x.double() / T
        m = xd.amax(1, keepdim=True)
        p = (xd - m).exp()
        p = p / p.sum(1, keepdim=True)
        hot = torch.zeros_like(p)
        hot[torch.arange(8, device="cuda"), ids] = 1.0
        g = (dlogp.double() / T)[:, None]
        ref = g * (hot - p)
        # the probability: SUM, and 2^-22 of its exponent; row 7 (and every row
        # with |lse| < 65536) also takes lse's half step, 2^-24 of it
        arg = torch.where(p > 0, (m - xd).clamp(max=1000) * 1.4427 * 2.0 ** -22, 0.0)
        half = torch.where(true.abs() < 65536, true.abs() * 2.0 ** -24, 0.0)[:, None]
        tol = g.abs() * (p * (R.SUM + arg + half) + (hot + p) * 2.0 ** -23) + ref.abs() * R.HALF[dtype] + 2.0 ** -125 * (1 + g.abs())
        near(got, ref, tol)
        same = x.clone()
        assert k.token_logprobs_grad(same, ids, lse, dlogp, temperature=T, out=same) is same and torch.equal(same, got)
        loss, lp2, dx = k.policy_loss(x, ids, None, -dlogp, temperature=T)  # r = 1: the same gradient
        assert torch.equal(lp2, logp)
        near(dx, ref, tol)
    # half of a row, with the whole row's lse
    x = (torch.randn(1, 2000, device="cuda", generator=gen(5)) + 2.0 ** 17).float()
    x[:, 1000:] += 4.0  # (so that the whole row's lse is 4 above the half's: 2^17 has steps of 2^-6)
    ids = torch.tensor([3], device="cuda")
    one = torch.ones(1, device="cuda")
    _, lse = k.token_logprobs(x, ids)
    got = k.token_logprobs_grad(x[:, :1000], ids, lse, one)
    ref, tol = R.grad(x[:, :1000], ids, 1.0, lse.double(), one.double(), F32)
    near(got, ref, tol)
    x[:, :1000] = -math.inf
    got = k.token_logprobs_grad(x[:, :1000], ids, lse, one)
    assert got[0, 3] == 1 and not bool(got[0, :3].any()) and not bool(got[0, 4:].any())


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("B", [3, 20, 50, 100])
def test_w4_scales_and_zero_points_at_any_address(B, g):
    """Rows of scales and zero points that allow wide loads and the same
    values at odd addresses: equal bits, and the definition's."""
    from mstar_rs_b200 import kernel as k

    V = 700
    for d in (1024, 2048, 1024 + 128):
        hidden = torch.randn(B, d, device="cuda", generator=gen(d)).to(BF16)
        for stype in (BF16, F32):
            codes, scales, zeros = w4_inputs(V, d, g, stype, True, B + d)

            def moved(t, by):
                flat = torch.empty(t.numel() + by, device="cuda", dtype=t.dtype)
                flat[by:] = t.flatten()
                return flat[by:].view(t.shape)

            for z in (zeros, None):
                out = k.lmhead_logits_w4(hidden, codes, scales, zeros=z)
                ref, tol = R.head(hidden, codes, scales, z, F32, parts=16)
                near(out, ref, tol)
                for by in (1, 2):
                    other = k.lmhead_logits_w4(hidden, codes, moved(scales, by), zeros=None if z is None else moved(z, by))
                    assert torch.equal(out, other)


@pytest.mark.parametrize("V,d", [(300, 256), (1302, 1280), (4099, 1024), (12000, 1024), (33000, 512)])
def test_w4_chunks_of_rows(V, d):
    """Batches around every chunk's width, over matrices of few and many
    units, against the definition; nothing beyond their rows and columns is
    written."""
    from mstar_rs_b200 import kernel as k

    codes, scales, zeros = w4_inputs(V, d, 64, BF16, True, V)
    hidden = torch.randn(256, d, device="cuda", generator=gen(d)).to(BF16)
    ref, tol = R.head(hidden, codes, scales, zeros, F32, parts=16)
    for B in (15, 16, 17, 31, 33, 48, 63, 65, 127, 129, 191, 193, 255, 256):
        rows = torch.arange(256, device="cuda")[-B:]
        out = torch.full((B + 1, V + 3), 7.0, device="cuda")
        got = k.lmhead_logits_w4(hidden[rows], codes, scales, zeros=zeros, out=out[:B, :V])
        near(got, ref[rows], tol[rows])
        assert bool((out[B] == 7).all()) and bool((out[:, V:] == 7).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_policy_loss_leaves_lse(dtype):
    """The C entry's lse is token_logprobs' (0 for padding rows)."""
    import ctypes

    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel as k

    n, V = 5, 777
    x = torch.randn(n, V, device="cuda", generator=gen(1)).to(dtype)
    x[2] = -math.inf
    ids = torch.tensor([3, -1, 4, V, 5], device="cuda")
    adv = torch.ones(n, device="cuda")
    loss, logp, lse = (torch.full((n,), 9.0, device="cuda") for _ in range(3))
    p = N.PolicyParams(x.data_ptr(), N.DTYPE_F32 if dtype == F32 else N.DTYPE_BF16, n, V, 0, V, ids.data_ptr(), None, None,
                       adv.data_ptr(), None, 1.0, 0.2, 0.2, 0.0, loss.data_ptr(), logp.data_ptr(), lse.data_ptr(), None,
                       0, None)
    k._call(x.device, "mstar_policy_loss", ctypes.byref(p))
    want_logp, want = k.token_logprobs(x, ids)
    assert torch.equal(lse, torch.where((ids >= 0) & (ids < V), want, 0.0)) and torch.equal(logp, want_logp)


@pytest.mark.parametrize("V,d", [(1302, 1280), (4099, 1024), (33000, 512)])
def test_w4_one_workspace_for_all_batches(V, d):
    """The largest batch's scratch, full of ones before each call, serves the
    smaller batches: the same bits as with fresh scratch."""
    from mstar_rs_b200 import kernel as k

    codes, scales, _ = w4_inputs(V, d, 64, BF16, False, V)
    hidden = torch.randn(200, d, device="cuda", generator=gen(d)).to(BF16)
    ws = k.lmhead_w4_workspace(200, V, d, "cuda")
    for B in (200, 129, 128, 65, 64, 33, 16, 1):
        ws.fill_(255)
        got = k.lmhead_logits_w4(hidden[:B], codes, scales, workspace=ws)
        assert torch.equal(got, k.lmhead_logits_w4(hidden[:B], codes, scales))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5, 1000, 40000])
def test_rows_without_a_number(V, dtype):
    """Rows of NaN alone, and of NaN among masked ids, are NaN and not empty:
    their log-probabilities, losses and gradients say so.  Padding rows among
    them stay zero and empty rows empty."""
    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel

    x = torch.full((7, V), -math.inf, device="cuda").to(dtype)
    x[0] = math.nan
    x[1, V - 1] = math.nan             # behind the aligned vectors, or in the last of them
    x[2, 0] = math.nan
    x[3] = torch.finfo(dtype).min
    x[3, 1] = math.nan                 # beside the type's lowest value
    x[4] = math.nan                    # padding
    x[6, V // 2] = math.nan            # (row 5 is empty)
    ids = torch.tensor([2, 2, 0, 2, -1, 2, V // 2], device="cuda")
    nan = torch.tensor([True, True, True, True, False, False, True], device="cuda")
    for T in (1.0, 1e-5, 1e5):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        logp, lse = kernel.token_logprobs(x[nan], ids[nan], temperature=T, status=status)
        assert status.item() == 0 and bool(logp.isnan().all()) and bool(lse.isnan().all())
        logp, lse = kernel.token_logprobs(x, ids, temperature=T)
        assert torch.equal(logp.isnan(), nan) and logp[4] == 0 and logp[5] == -math.inf and lse[5] == -math.inf
        one = torch.ones(7, device="cuda")
        g = kernel.token_logprobs_grad(x, ids, lse, one, temperature=T)
        assert bool(g[nan].isnan().all()) and not bool(g[4:6].any())
        for old in (None, one):
            for adv in (one, -one, 0 * one):
                status.zero_()
                loss, lp, dx = kernel.policy_loss(x, ids, old, adv, ref_logp=one, kl_coef=0.1, temperature=T, status=status)
                assert status.item() == N.STATUS_EMPTY
                assert torch.equal(lp.isnan(), nan) and torch.equal(loss.isnan(), nan) and not bool(loss[4:6].any())
                assert bool(dx[nan].isnan().all()) and not bool(dx[4:6].any())
                value = kernel.policy_loss(x, ids, old, adv, ref_logp=one, kl_coef=0.1, temperature=T, grad=False)[0]
                assert torch.equal(value.isnan(), nan)


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("V,d", [(2000, 128), (70000, 384), (9001, 640), (40000, 1152)])
def test_w4_odd_numbers_of_blocks(V, d, g):
    """Widths of an odd number of 128-column blocks, where the blocks of one
    tile end in the middle of a stage, over one and many tiles per CTA."""
    from mstar_rs_b200 import kernel as k

    codes, scales, zeros = w4_inputs(V, d, g, BF16, True, V)
    hidden = torch.randn(64, d, device="cuda", generator=gen(d)).to(BF16)
    ref, tol = R.head(hidden, codes, scales, zeros, F32, parts=16)
    for B in (1, 16, 17, 32, 64):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        first = k.lmhead_logits_w4(hidden[:B], codes, scales, zeros=zeros, status=status)
        near(first, ref[:B], tol[:B])
        for _ in range(3):
            assert torch.equal(first, k.lmhead_logits_w4(hidden[:B], codes, scales, zeros=zeros, status=status))
        assert status.item() == 0


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("B,V,d", [(1, 70000, 384), (16, 4099, 1024), (32, 20011, 640), (64, 20011, 1024), (128, 9001, 896),
                                   (200, 9001, 512)])
def test_w4_withheld_copy_runs_out(B, V, d, g):
    """Each CTA's last copy of hidden rows is never issued (no bad address, no
    copy in flight): the waits on it give up after their limit, the call
    returns and sets the status bit, and the next call with the same scratch
    is right."""
    from mstar_rs_b200 import _native as N
    from mstar_rs_b200 import kernel as k

    codes, scales, zeros = w4_inputs(V, d, g, BF16, True, V)
    hidden = torch.randn(B, d, device="cuda", generator=gen(d)).to(BF16)
    logits = torch.zeros(B, V, device="cuda")
    ids = torch.zeros(B, dtype=torch.int64, device="cuda")
    ws = k.lmhead_w4_workspace(B, V, d, "cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(zeros=zeros, status=status, workspace=ws, out_ids=ids, uniforms=torch.full((B,), 0.5, device="cuda"))
    k.lmhead_step_w4(hidden, codes, scales, logits, flags=N.FLAG_TEST_WITHHOLD, **kw)
    torch.cuda.synchronize()
    assert status.item() == 1
    status.zero_()
    k.lmhead_step_w4(hidden, codes, scales, logits, **kw)
    assert status.item() == 0
    ref, tol = R.head(hidden, codes, scales, zeros, F32, parts=16)
    near(logits, ref, tol)


@pytest.mark.parametrize("n,V", [(4, 3001), (2, 70000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_keeps_the_probabilities_of_large_lse(dtype, n, V):
    """The gradient's probabilities at every size of lse: its rounding to 32
    bits (2^-24 of itself) costs f32 gradients at most 2^-16 and bf16 ones, whose
    own half step is 2^-8, 2^-9; larger ones are summed anew."""
    from mstar_rs_b200 import kernel as k

    limit = 256 if dtype == F32 else 2 ** 15
    for T, shift in ((1.0, 150.0), (1.0, -1e4), (0.01, 0.0), (1.0, 300.0), (1.0, 20000.0), (0.5, -30000.0), (1.0, 65000.0)):
        x = (torch.randn(n, V, device="cuda", generator=gen(n)) + shift).to(dtype)
        x[1, 1::3] = -math.inf
        ids = torch.randint(0, V // 3, (n,), device="cuda", generator=gen(1)) * 3
        dlogp = torch.randn(n, device="cuda", generator=gen(2))
        _, lse = k.token_logprobs(x, ids, temperature=T)
        got = k.token_logprobs_grad(x, ids, lse, dlogp, temperature=T)
        xd = x.double() / T
        m = xd.amax(1, keepdim=True)
        p = (xd - m).exp()
        s = p.sum(1, keepdim=True)
        p, true = p / s, (m + s.log())[:, 0]
        hot = torch.zeros_like(p)
        hot[torch.arange(n, device="cuda"), ids] = 1.0
        g = (dlogp.double() / T)[:, None]
        ref = g * (hot - p)
        arg = torch.where(p > 0, (m - xd).clamp(max=1000) * 1.4427 * 2.0 ** -22, 0.0)
        half = torch.where(true.abs() < limit, true.abs() * 2.0 ** -24, 0.0)[:, None]
        tol = g.abs() * (p * (R.SUM + arg + half) + (hot + p) * 2.0 ** -23) + ref.abs() * R.HALF[dtype] + 2.0 ** -125 * (1 + g.abs())
        near(got, ref, tol)
        same = x.clone()
        assert k.token_logprobs_grad(same, ids, lse, dlogp, temperature=T, out=same) is same and torch.equal(same, got)


def test_w4_outputs_apart_from_their_inputs():
    """An output that lies on what the call reads is refused before anything is
    launched; one right beside it is not."""
    from mstar_rs_b200 import kernel as k

    V, d, B = 64, 128, 4
    # one buffer: logits between the hidden rows and codes, scales and zeros
    buf = torch.zeros(1 << 16, device="cuda", dtype=torch.uint8)
    at, place = 0, {}
    for name, n in (("hidden", B * d * 2), ("out", B * V * 4), ("codes", V * d // 2), ("scales", V * 4 * 4), ("zeros", V * 4)):
        place[name] = at
        at += n

    def view(name, dtype, *shape, move=0):
        n = math.prod(shape) * torch.tensor([], dtype=dtype).element_size()
        return buf[place[name] + move:place[name] + move + n].view(dtype).view(*shape)

    hidden, codes = view("hidden", BF16, B, d), view("codes", torch.uint8, V, d // 2)
    scales, zeros = view("scales", F32, V, 4), view("zeros", torch.uint8, V, 4)
    hidden.copy_(torch.randn(B, d, device="cuda", generator=gen(1)))
    for t, u in zip((codes, scales, zeros), w4_inputs(V, d, 32, F32, True, 2)):
        t.copy_(u)
    keep = buf.clone()
    ids = torch.tensor([3, -1], device="cuda")
    step = dict(zeros=zeros, out_ids=torch.zeros(B, dtype=torch.int64, device="cuda"),
                uniforms=torch.full((B,), 0.5, device="cuda"))
    for name, move, what in (("out", -4, "hidden"), ("out", 16, "codes"), ("codes", 0, "codes"), ("scales", -16, "codes"),
                             ("scales", 16, "scales"), ("zeros", 64, "zeros")):
        with pytest.raises(ValueError, match=what):
            k.lmhead_logits_w4(hidden, codes, scales, zeros=zeros, out=view(name, F32, B, V, move=move))
        with pytest.raises(ValueError, match=what):
            k.lmhead_step_w4(hidden, codes, scales, view(name, F32, B, V, move=move), **step)
    for name, move, what in (("codes", 64, "codes"), ("scales", 32, "scales"), ("zeros", 64, "zeros")):
        with pytest.raises(ValueError, match=what):
            k.embed_tokens_w4(ids, codes, scales, zeros=zeros, out=view(name, F32, 2, d, move=move))
    assert torch.equal(buf, keep)
    out = view("out", F32, B, V)
    k.lmhead_logits_w4(hidden, codes, scales, zeros=zeros, out=out)
    assert torch.equal(out, k.lmhead_logits_w4(hidden.clone(), codes.clone(), scales.clone(), zeros=zeros.clone()))
    row = view("out", F32, 2, d)
    k.embed_tokens_w4(ids, codes, scales, zeros=zeros, out=row)
    assert torch.equal(row, k.embed_tokens_w4(ids, codes.clone(), scales.clone(), zeros=zeros.clone(), dtype=F32))


def test_w4_outputs_of_another_type():
    """A type that the logits or rows cannot have is a TypeError, as in every
    other call."""
    from mstar_rs_b200 import kernel as k

    codes, scales, zeros = w4_inputs(64, 128, 32, F32, True, 1)
    for dt in (torch.float16, torch.float64, torch.int32):
        with pytest.raises(TypeError):
            k.lmhead_logits_w4(torch.zeros(4, 128, device="cuda", dtype=BF16), codes, scales, dtype=dt)
        with pytest.raises(TypeError):
            k.embed_tokens_w4(torch.zeros(4, dtype=torch.int64, device="cuda"), codes, scales, dtype=dt)
        with pytest.raises(TypeError):
            k.embed_tokens_grad(torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, 8, device="cuda"), 9, dtype=dt)


@pytest.mark.parametrize("V,d", [(1, 1), (40, 3), (37, 64), (500, 501), (3000, 128)])
@pytest.mark.parametrize("ot", [BF16, F32])
def test_embed_grad_at_any_address(V, d, ot):
    """Outputs and bases that start off a 16-byte border, at the same place
    modulo 16 bytes and at different ones: the definition's values, and nothing
    before or behind the output is written."""
    from mstar_rs_b200 import kernel as k

    n = 2 * V + 5
    ids = torch.randint(-1, V + 1, (n,), device="cuda", generator=gen(V))
    dout = torch.randn(n, d, device="cuda", generator=gen(d)).to(BF16)
    base = torch.randn(V, d, device="cuda", generator=gen(3)).to(ot)
    fresh = {False: k.embed_tokens_grad(ids, dout, V, dtype=ot), True: k.embed_tokens_grad(ids, dout, V, base=base, dtype=ot)}
    for kind, got in fresh.items():
        ref, tol = R.embed_grad(ids, dout, V, 1.0, base if kind else None, ot)
        near(got, ref, tol)

    def at(places):
        buf = torch.full((V * d + 32,), 5.0, device="cuda").to(ot)
        return buf, buf[places:places + V * d].view(V, d)

    for i in range(0, 9):
        buf, out = at(i)
        k.embed_tokens_grad(ids, dout, V, out=out)
        assert torch.equal(out, fresh[False])
        assert bool((buf[:i] == 5).all()) and bool((buf[i + V * d:] == 5).all())
        for j in (i, i + 1, 8 - i):
            buf, out = at(i)
            keep, b = at(j)
            b.copy_(base)
            k.embed_tokens_grad(ids, dout, V, base=b, out=out)
            assert torch.equal(out, fresh[True]) and torch.equal(b, base)
            assert bool((buf[:i] == 5).all()) and bool((buf[i + V * d:] == 5).all())
        buf, out = at(i)
        out.copy_(base)
        k.embed_tokens_grad(ids, dout, V, base=out, out=out)
        assert torch.equal(out, fresh[True])
        assert bool((buf[:i] == 5).all()) and bool((buf[i + V * d:] == 5).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lmhead_step_w4_against_the_oracle(oracle_lib, dtype):
    """The one call at full size: its logits against the 4-bit definition, and
    the ids that the oracle takes from those logits."""
    import numpy as np

    from mstar_rs_b200 import kernel as k
    from mstar_rs_b200 import workloads as W

    B, V, d = 64, 151936, 2048
    case = W.qwen_mixed(seed=8, B=B, V=V)
    case.dtype = dtype
    kw = W.to_device(case)
    kw.pop("logits")
    codes, scales, z = w4_inputs(V, d, 128, BF16, True, 6)
    scales *= 4  # (logits of some units, so that the cuts of top_p and min_p are met)
    hidden = torch.randn(B, d, device="cuda", generator=gen(4)).to(BF16)
    tdt = BF16 if dtype == "bf16" else F32
    logits = torch.empty(B, V, dtype=tdt, device="cuda")
    ids = torch.zeros(B, dtype=torch.int64, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    k.lmhead_step_w4(hidden, codes, scales, logits, zeros=z, status=st, **kw, out_ids=ids)
    assert st.item() == 0
    for v in range(0, V, 30000):  # (in parts: the definition is in 64 bits)
        part = slice(v, min(V, v + 30000))
        ref, tol = R.head(hidden, codes[part], scales[part], z[part], tdt, parts=16)
        near(logits[:, part], ref, tol)
    case.logits = logits.float().cpu().numpy() if dtype == "f32" else logits.view(torch.int16).cpu().numpy().view(np.uint16)
    assert np.array_equal(ids.cpu().numpy(), oracle_lib.run(case)["ids"])


@pytest.mark.parametrize("stages,V", [(11, 700), (13, 2000), (17, 300), (19, 4099), (22, 1000), (23, 257), (37, 600)])
def test_w4_stages_without_a_near_divisor(stages, V):
    """Widths whose stages do not divide evenly over a tile's CTAs."""
    from mstar_rs_b200 import kernel as k

    for d in (stages * 256, stages * 256 - 128):
        codes, scales, zeros = w4_inputs(V, d, 64, F32, True, d)
        hidden = torch.randn(40, d, device="cuda", generator=gen(V)).to(BF16)
        ref, tol = R.head(hidden, codes, scales, zeros, F32, parts=16)
        for B in (1, 16, 40):
            out = k.lmhead_logits_w4(hidden[:B], codes, scales, zeros=zeros)
            near(out, ref[:B], tol[:B])
            assert torch.equal(out, k.lmhead_logits_w4(hidden[:B], codes, scales, zeros=zeros))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5000, 22357, 151936])
def test_rows_under_finite_masks(V, dtype):
    """Masks of every finite size over most of a row, in the front of it, the
    back or throughout, at every temperature: the ids left have the whole
    probability, masked ones none."""
    from mstar_rs_b200 import kernel as k

    n = 6
    for mask in (-1e4, -1e9, -1e10, -1e15, -1e25, -1e30, -1e35, torch.finfo(dtype).min):
        for T in (1.0, 0.3, 0.01, 1e-5, 1e5):
            G = gen(V)
            x = torch.randn(n, V, device="cuda", generator=G).to(dtype)
            hide = torch.rand(n, V, device="cuda", generator=G) < 0.999
            hide[1, :-9], hide[1, -9:] = True, False   # the front
            hide[2, :9], hide[2, 9:] = False, True     # the back
            hide[3] = True
            hide[3, V // 2] = False                    # all but one
            hide[4] = False
            hide[:, V // 3] = False
            x = torch.where(hide, mask, x.double()).to(dtype)
            ids = torch.full((n,), V // 3, device="cuda")
            logp, lse = k.token_logprobs(x, ids, temperature=T)
            _, rl, rp = R.rows(x, ids, T)
            near(lse, rl.clamp(-3.4028234e38, 3.4028234e38), R.SUM + rl.abs() * 2.0 ** -23)
            near(logp, rp, R.SUM + rp.abs() * 2.0 ** -23)
            one = torch.ones(n, device="cuda")
            loss, lp2, dx = k.policy_loss(x, ids, None, -one, temperature=T)  # r = 1, A = -1: loss 1, gradient of logp
            assert torch.equal(lp2, logp) and bool((loss == 1).all())
            g = k.token_logprobs_grad(x, ids, lse, one, temperature=T)
            xd = x.double() / T
            m = xd.amax(1, keepdim=True)
            p = (xd - m).exp()
            p = p / p.sum(1, keepdim=True)
            ref = -p / T
            ref[:, V // 3] += 1 / T
            arg = torch.where(p > 0, (m - xd).clamp(max=1000) * 1.4427 * 2.0 ** -22, 0.0)
            limit = 256 if dtype == F32 else 2 ** 15
            half = torch.where(rl.abs() < limit, rl.abs() * 2.0 ** -24, 0.0)[:, None]
            # (the id's own place is off by what its probability and 1 are)
            tol = (p * (R.SUM + arg) + p * 2.0 ** -22) / T + ref.abs() * R.HALF[dtype] + 2.0 ** -125 * (1 + 1 / T)
            tol[:, V // 3] += 2.0 ** -23 / T
            near(dx, ref, tol)
            near(g, ref, tol + p * half / T)
