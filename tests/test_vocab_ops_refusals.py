"""CPU: what the vocabulary operators refuse, in the front end and behind the
C ABI, before anything is launched; and the 4-bit format's plain helper."""
import ctypes

import pytest
import torch

from mstar_rs_b200 import _native as N
from mstar_rs_b200 import kernel

INV = N.ERR_INVALID


@pytest.fixture(scope="module")
def L():
    from mstar_rs_b200 import build

    build.build()
    return N.lib()


def refused(L, rc, word):
    assert rc == INV
    assert word in L.mstar_sampler_last_error().decode(), L.mstar_sampler_last_error()


def w4(**kw):
    f = dict(codes=0x1000, scales=0x2000, zeros=None, V=100, d=256, group=128, scale_dtype=N.DTYPE_F32)
    f.update(kw)
    return N.W4(**f)


@pytest.mark.parametrize("kw,word", [
    (dict(codes=None), "codes"), (dict(scales=None), "scales"), (dict(codes=0x1008), "16-byte"),
    (dict(scales=0x2002), "aligned"), (dict(scale_dtype=5), "scale_dtype"), (dict(group=48), "group"),
    (dict(d=192), "multiple of group"), (dict(V=0), "V must"), (dict(d=0), "multiple of group")])
def test_w4_matrix(L, kw, word):
    w = w4(**kw)
    refused(L, L.mstar_lmhead_logits_w4(0x1000, 256, 1, ctypes.byref(w), 0x3000, 0, 100, 0x4000, 1 << 30, None, None), word)
    refused(L, L.mstar_embed_tokens_w4(0x1000, 1, ctypes.byref(w), 1.0, 0x3000, 0, None, None), word)


def test_w4_head(L):
    w = w4()
    call = lambda hidden=0x1000, ldh=256, B=1, out=0x3000, dt=0, ld=100, ws=0x4000, n=1 << 30: L.mstar_lmhead_logits_w4(  # noqa: E731
        hidden, ldh, B, ctypes.byref(w), out, dt, ld, ws, n, None, None)
    refused(L, call(hidden=None), "hidden")
    refused(L, call(hidden=0x1001), "aligned")
    refused(L, call(ldh=255), "ld_hidden")
    refused(L, call(B=0), "B must")
    refused(L, call(B=257), "B must")
    refused(L, call(out=None), "logits")
    refused(L, call(out=0x3002), "aligned")
    refused(L, call(dt=3), "dtype")
    refused(L, call(ld=99), "ld must")
    refused(L, call(ws=None), "workspace")
    refused(L, call(ws=0x4010), "256-byte")
    need = L.mstar_lmhead_w4_workspace_bytes(1, 100, 256)
    assert need > 0
    refused(L, call(n=need - 1), "too small")
    refused(L, L.mstar_lmhead_logits_w4(0x1000, 256, 1, None, 0x3000, 0, 100, 0x4000, 1 << 30, None, None), "w is NULL")
    for bad in ((0, 100, 256), (257, 100, 256), (1, 0, 256), (1, 100, 100), (1, 100, 0)):
        assert L.mstar_lmhead_w4_workspace_bytes(*bad) == -1
    p = N.Params()
    p.V = 99
    refused(L, L.mstar_sampler_lmhead_step_w4(ctypes.byref(p), 0x1000, 256, ctypes.byref(w), 0x4000, 1 << 30, None, None), "V rows")
    p.V = 100  # the step's own checks come before the projection
    refused(L, L.mstar_sampler_lmhead_step_w4(ctypes.byref(p), 0x1000, 256, ctypes.byref(w), 0x4000, 1 << 30, None, None), "logits")
    assert L.mstar_sampler_lmhead_step_w4(None, 0x1000, 256, ctypes.byref(w), 0x4000, 1 << 30, None, None) == INV


def test_lookup(L):
    call = lambda ids=0x1000, n=4, table=0x2000, dt=0, V=10, d=8, ld=8, out=0x3000, odt=0: L.mstar_embed_tokens(  # noqa: E731
        ids, n, table, dt, V, d, ld, 1.0, out, odt, None, None)
    refused(L, call(ids=None), "ids")
    refused(L, call(out=None), "out")
    refused(L, call(table=None), "table")
    refused(L, call(n=0), "N must")
    refused(L, call(n=1 << 29), "N must")
    refused(L, call(V=0), "V must")
    refused(L, call(d=0), "d must")
    refused(L, call(ld=7), "ld must")
    refused(L, call(dt=2), "dtype")
    refused(L, call(odt=2), "out_dtype")
    refused(L, call(table=0x2002), "aligned")
    refused(L, call(out=0x3001), "aligned")
    w = w4()
    refused(L, L.mstar_embed_tokens_w4(0x1000, 4, ctypes.byref(w), 1.0, 0x3008, 1, None, None), "16-byte")


def test_lookup_gradient(L):
    call = lambda ids=0x1000, n=4, dout=0x2000, dt=0, ld=8, V=10, d=8, base=None, out=0x3000, odt=0, ws=0x4000, nb=1 << 30: \
        L.mstar_embed_tokens_grad(ids, n, dout, dt, ld, V, d, 1.0, base, out, odt, ws, nb, None, None)  # noqa: E731
    for kw in (dict(ids=None), dict(dout=None), dict(out=None), dict(ws=None)):
        refused(L, call(**kw), "NULL")
    refused(L, call(n=0), "N must")
    refused(L, call(n=(1 << 24) + 1), "N must")
    refused(L, call(V=(1 << 21) + 1), "V must")
    refused(L, call(d=65537, ld=65537), "d must")
    refused(L, call(ld=7), "ld must")
    refused(L, call(dt=2), "dtype")
    refused(L, call(odt=-1), "out_dtype")
    refused(L, call(dout=0x2001), "aligned")
    refused(L, call(base=0x3001), "aligned")
    refused(L, call(ws=0x4001), "256-byte")
    need = L.mstar_embed_grad_workspace_bytes(4, 10, 8)
    refused(L, call(nb=need - 1), "too small")
    for bad in ((0, 10, 8), (4, 0, 8), (4, 10, 0), (1 << 25, 10, 8), (4, 1 << 22, 8), (4, 10, 1 << 17)):
        assert L.mstar_embed_grad_workspace_bytes(*bad) == -1


def test_rows(L):
    call = lambda x=0x1000, dt=0, n=2, V=10, ld=10, ids=0x2000, T=1.0, lp=0x3000: L.mstar_token_logprobs(  # noqa: E731
        x, dt, n, V, ld, ids, T, lp, None, None, None)
    refused(L, call(x=None), "logits")
    refused(L, call(ids=None), "ids")
    refused(L, call(lp=None), "logp")
    refused(L, call(dt=9), "dtype")
    refused(L, call(n=0), "N must")
    refused(L, call(V=0), "V must")
    refused(L, call(ld=9), "ld must")
    refused(L, call(x=0x1002), "aligned")
    for T in (0.0, -1.0, 1e-6, 1e6, float("nan"), float("inf")):
        refused(L, call(T=T), "temperature")
    g = lambda lse=0x3000, d=0x4000, out=0x5000, ld=10: L.mstar_token_logprobs_grad(  # noqa: E731
        0x1000, 0, 2, 10, 10, 0x2000, 1.0, lse, d, out, ld, None)
    refused(L, g(lse=None), "lse")
    refused(L, g(d=None), "dlogp")
    refused(L, g(out=None), "dlogits")
    refused(L, g(out=0x5001), "aligned")
    refused(L, g(ld=9), "ld_dlogits")


def test_policy(L):
    def call(**kw):
        f = dict(logits=0x1000, dtype=0, N=2, V=10, ld=10, ids=0x2000, old_logp=None, ref_logp=None, advantages=0x3000,
                 weights=None, temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, loss=0x4000, logp=0x5000,
                 lse=None, dlogits=None, ld_dlogits=0, status=None)
        f.update(kw)
        return L.mstar_policy_loss(ctypes.byref(N.PolicyParams(**f)), None)

    assert L.mstar_policy_loss(None, None) == INV
    refused(L, call(advantages=None), "advantages")
    refused(L, call(loss=None), "loss")
    refused(L, call(logp=None), "logp")
    refused(L, call(clip_low=1.5), "clip_low")
    refused(L, call(clip_low=float("nan")), "clip_low")
    refused(L, call(clip_high=-0.1), "clip_high")
    refused(L, call(kl_coef=-1.0), "kl_coef")
    refused(L, call(kl_coef=float("nan")), "kl_coef")
    refused(L, call(kl_coef=0.1), "ref_logp")
    refused(L, call(dlogits=0x6000, ld_dlogits=9), "ld_dlogits")
    refused(L, call(dlogits=0x6002, ld_dlogits=10), "aligned")
    refused(L, call(temperature=0.0), "temperature")


@pytest.mark.parametrize("struct,ctype", [(N.W4, "mstar_w4_t"), (N.PolicyParams, "mstar_policy_params_t")])
def test_struct_layouts_match_the_header(tmp_path, struct, ctype):
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [f[0] for f in struct._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"mstar_sampler.h\"\nint main(void){\n"
    src += f'printf("%zu\\n", sizeof({ctype}));\n'
    src += "".join(f'printf("%zu\\n", offsetof({ctype}, {n}));\n' for n in names) + "return 0;}\n"
    c, exe = tmp_path / "t.c", tmp_path / "t"
    c.write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), "-o", str(exe), str(c)])
    out = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert out[0] == ctypes.sizeof(struct)
    assert [getattr(struct, n).offset for n in names] == out[1:]


def test_front_end_has_no_cpu_path():
    x, ids = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int64)
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1)
    f = torch.zeros(2)
    for call in (lambda: kernel.token_logprobs(x, ids), lambda: kernel.token_logprobs_grad(x, ids, f, f),
                 lambda: kernel.policy_loss(x, ids, f, f), lambda: kernel.embed_tokens(ids, x),
                 lambda: kernel.embed_tokens_grad(ids, x, 5), lambda: kernel.embed_tokens_w4(ids, codes, scales),
                 lambda: kernel.lmhead_logits_w4(x.bfloat16(), codes, scales)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("group,zero_points,sdt", [(32, False, torch.float32), (64, True, torch.bfloat16), (128, True, torch.float32)])
def test_quantize_w4(group, zero_points, sdt):
    """A quantised weight is off by at most half a step of its group, and by
    the codes that the range's ends clamp (without zero points, +7.5 steps)."""
    from tests import vocab_ref as R

    w = torch.randn(20, 256, generator=torch.Generator().manual_seed(3))
    w[3] = 0.0
    w[4] = w[4].abs()
    codes, scales, zeros = kernel.quantize_w4(w, group, zero_points=zero_points, scale_dtype=sdt)
    assert codes.shape == (20, 128) and codes.dtype == torch.uint8
    assert scales.shape == (20, 256 // group) and scales.dtype == sdt and (zeros is not None) == zero_points
    back = R.dequant(codes, scales, zeros)
    step = scales.double().repeat_interleave(group, 1)
    # without zero points 7.5 steps reach the largest value, and code 15 is 7 of
    # them; with them the zero point's own rounding moves the range by half a
    # step.  A bf16 scale is off by 2^-8, up to 15 steps of it at the far end.
    limit = 1.0 + (15 * 2.0 ** -8 if sdt == torch.bfloat16 else 1e-5)
    assert bool(((back - w.double()).abs() <= step * limit + 1e-12).all())
    assert bool((back[3] == 0).all())
    for bad in (dict(group_size=48), dict(group_size=96)):
        with pytest.raises(ValueError):
            kernel.quantize_w4(w, **bad)
    with pytest.raises(ValueError):
        kernel.quantize_w4(w[0])
    with pytest.raises(TypeError):
        kernel.quantize_w4(w, scale_dtype=torch.float16)


@pytest.mark.parametrize("V,d", [(300, 256), (4099, 1024), (2048, 4096), (32000, 2048), (151936, 2048)])
def test_w4_workspace_of_a_larger_batch_serves_smaller_ones(V, d):
    lib = N.lib()
    sizes = [lib.mstar_lmhead_w4_workspace_bytes(B, V, d) for B in range(1, 257)]
    assert sizes[0] > 0 and all(a <= b for a, b in zip(sizes, sizes[1:]))


@pytest.mark.parametrize("d", [1, 513, 1024, 2048, 5000, 65536])
def test_embed_grad_workspace_of_more_tokens_serves_fewer(d):
    lib = N.lib()
    counts = list(range(1, 4000)) + list(range(4000, 400000, 37))
    sizes = [lib.mstar_embed_grad_workspace_bytes(n, 4099, d) for n in counts]
    assert sizes[0] > 0 and all(a <= b for a, b in zip(sizes, sizes[1:]))


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantize_w4_of_views(zero_points):
    """A transposed weight, and one inside a wider matrix, give what their
    copies give, in the contiguous rows that the calls ask for."""
    wide = torch.randn(256, 300, generator=torch.Generator().manual_seed(5))
    for w in (wide.t()[:, :128], wide[3:50, 7:135], wide.bfloat16().t()[::2, 64:192]):
        got = kernel.quantize_w4(w, 32, zero_points=zero_points)
        want = kernel.quantize_w4(w.contiguous(), 32, zero_points=zero_points)
        for a, b in zip(got, want):
            assert (a is None and b is None) or (a.is_contiguous() and torch.equal(a, b))
