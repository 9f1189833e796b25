"""Block operators (ops.py) at the edges of what their documentation allows.  Formulas, cases and tolerances: test_block_ops.py."""
import ctypes as C
import math
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from conftest import PKG
from test_block_ops import E, attention_case, half_step, native, norm64, norm_case, ops, rounding, within

REPO = Path(__file__).resolve().parent.parent

EMPTY_WORKSPACES = """
import ctypes as C, importlib
n = importlib.import_module("%s._native")
lib, P = n.load(), 0x1000
for size in (dict(batch=1, seq=0), dict(batch=0, seq=1), dict(batch=0, seq=0)):
    for more in (dict(), dict(d_scale=P, scale_stride=8), dict(d_scale=P), dict(d_y=P, d_gate=P, gate_stride=8, d_shift=P)):
        d = n.GatedNormDesc(**size, dim=8, post=0, pre=2, residual_scale=1.0, eps=1e-5, d_x=P, d_weight=P, **more)
        for g in (n.GatedNormGrads(d_gx=P), n.GatedNormGrads(d_gx=P, d_gweight=P), n.GatedNormGrads(d_gscale=P if "d_scale" in more else 0)):
            print(lib.cmdi_gated_norm_vjp_workspace(C.byref(d), C.byref(g)), flush=True)
""" % PKG


def test_gated_norm_workspace_without_rows():
    """No rows need no workspace (in a process of its own: a division by zero would end it)."""
    run = subprocess.run([sys.executable, "-c", EMPTY_WORKSPACES], cwd=REPO, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and run.stdout.split() == ["0"] * 36, (run.returncode, run.stdout, run.stderr)
    n = native()
    d = n.GatedNormDesc(batch=0, seq=1, dim=0, post=0, pre=2, residual_scale=1.0, eps=1e-5)
    assert n.load().cmdi_gated_norm_vjp_workspace(C.byref(d), C.byref(n.GatedNormGrads())) == -1      # the other checks come first


LAUNCHES = """
#include <cstdio>
#include "launches.hpp"
int main() {
    long long blocks, whole;
    int threads;
    while (std::scanf("%lld %d %lld", &blocks, &threads, &whole) == 3) {
        cmdi::in_launches(blocks, threads, whole, [](int64_t first, unsigned n) { std::printf("%lld:%u ", (long long)first, n); return 0; });
        std::printf("\\n");
    }
}
"""


def test_launches_cover_all_blocks_and_stay_below_2_to_32_threads(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no C++ compiler")
    (tmp_path / "l.cpp").write_text(LAUNCHES)
    subprocess.run([cxx, "-std=c++17", "-I", str(REPO / PKG / "csrc"), str(tmp_path / "l.cpp"), "-o", str(tmp_path / "l")], check=True)
    cases = [(b, t, w) for t in (128, 256, 512, 1024) for w in (1, 3, 256)
             for b in (w, 5 * w, (1 << 21) // w * w, ((1 << 22) // w + 1) * w, ((1 << 31) // w) * w, ((1 << 31) - 1) * w)]
    out = subprocess.run([str(tmp_path / "l")], input="\n".join(f"{b} {t} {w}" for b, t, w in cases), capture_output=True, text=True, check=True).stdout
    for (b, t, w), line in zip(cases, out.splitlines()):
        parts = [tuple(map(int, p.split(":"))) for p in line.split()]
        assert sum(n for _, n in parts) == b and parts[0][0] == 0, (b, t, w)
        for (f, n), (g, _) in zip(parts, parts[1:]):
            assert n % w == 0 and f + n // w == g, (b, t, w)
        assert max(n for _, n in parts) * t < 1 << 32, (b, t, w)
    assert len(out.splitlines()) == len(cases)


@pytest.mark.gpu
def test_gated_norm_more_samples_than_a_launch_has_blocks():
    """2^23 + 5 samples of one row: the rows' pass takes two launches, the joins of their column sums five."""
    b, d = (1 << 23) + 5, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, y, gr, gh, scale, shift, gate = rnd(b, 1, d), rnd(b, 1, d).abs(), rnd(b, 1, d).abs(), rnd(b, 1, d), rnd(b, d), rnd(b, d), rnd(d)
    kw = dict(gate=gate, pre="rms")
    r, h = ops().gated_norm_fwd(x, y, scale=scale, shift=shift, **kw)
    got = ops().gated_norm_vjp(gr, gh, x, y, scale=scale, shift=shift, **kw)
    for at in (0, (1 << 21) - 2, (1 << 22) - 2, (1 << 23) - 2):
        p = slice(at, at + 7)
        r2, h2 = ops().gated_norm_fwd(x[p], y[p], scale=scale[p], shift=shift[p], **kw)
        assert torch.equal(r[p], r2) and torch.equal(h[p], h2), at
        part = ops().gated_norm_vjp(gr[p], gh[p], x[p], y[p], scale=scale[p], shift=shift[p], **kw)
        for n in ("x", "y", "scale", "shift"):
            assert torch.equal(got[n][p], part[n]), (n, at)
    # dr = gr where h has no gradient: dgate = sum gr y, all terms positive; 16 slices add 2^19 samples each one after another, then each other
    got = ops().gated_norm_vjp(gr, None, x, y, scale=scale, shift=shift, **kw, wanted=("gate", "scale"))
    want = (gr.double() * y.double()).sum((0, 1))
    within(got["gate"], want, ((1 << 19) + 144) * E * want, "gate")
    assert not got["scale"].any()


def test_refusal_of_a_lost_gradient():
    o, t = ops(), torch.zeros(2, requires_grad=True)
    with pytest.raises(native().NativeError, match="no backward pass"):
        o._no_backward("f", None, torch.zeros(2), t)
    with torch.no_grad():
        o._no_backward("f", None, t)
    o._no_backward("f", None, t.detach())


@pytest.mark.gpu
def test_8_bit_layer_refuses_every_call_that_would_lose_a_gradient():
    o, err = ops(), native().NativeError
    i8 = lambda *s: torch.ones(*s, dtype=torch.int8, device="cuda")  # noqa: E731
    one = lambda *s: torch.ones(*s, device="cuda")  # noqa: E731
    leaf = lambda *s: one(*s).requires_grad_()  # noqa: E731
    a, w, x = i8(3, 128), i8(5, 128), one(3, 128)
    calls = [lambda: o.quantize_rows(leaf(3, 100)),
             lambda: o.gemm_i8(a, leaf(3), w, one(5)), lambda: o.gemm_i8(a, one(3), w, leaf(5)), lambda: o.gemm_i8(a, one(3), w, one(5), leaf(5)),
             lambda: o.gemm_i8(a, one(3), w, one(5), epi="resid", resid=leaf(3, 5)),
             lambda: o.linear_i8(leaf(3, 128), w, one(5)), lambda: o.linear_i8(x, w, leaf(5)), lambda: o.linear_i8(x, w, one(5), leaf(5)),
             lambda: o.linear_i8(x, w, one(5), epi="resid", resid=leaf(3, 5))]
    for i, call in enumerate(calls):
        with pytest.raises(err, match="no backward pass"):
            call()
            pytest.fail(f"call {i} was accepted")
        with torch.no_grad():
            call()
    for want, got in zip(o.quantize_rows(one(3, 100)), o.quantize_rows(leaf(3, 100).detach())):
        assert torch.equal(want, got)


def test_refusal_of_a_lost_tangent():
    o, t = ops(), torch.zeros(2)
    with forward_ad.dual_level():
        o._no_tangent("f", None, t)
        with pytest.raises(native().NativeError, match="forward-mode"):
            o._no_tangent("f", None, t, forward_ad.make_dual(t, torch.ones(2)))
    o._no_tangent("f", None, t)


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """A tensor with a tangent, whether it requires a gradient or not, gives no result without one."""
    o, err = ops(), native().NativeError
    one = lambda *s: torch.ones(*s, device="cuda")  # noqa: E731
    half = lambda *s: one(*s).half()  # noqa: E731
    x, w8 = one(1, 2, 64), torch.ones(5, 128, dtype=torch.int8, device="cuda")
    a8, q, k, own = torch.ones(2, 128, dtype=torch.int8, device="cuda"), half(1, 1, 2, 64), half(4, 2, 64), half(1, 3, 2, 64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: o.gated_norm(dual(x)), lambda: o.gated_norm(dual(one(1, 2, 64).requires_grad_())), lambda: o.gated_norm(x, dual(x)),
                 *(lambda n=n: o.gated_norm(x, x, post="layer", **{n: dual(one(64))}) for n in o._PARAMS),
                 lambda: o.gated_norm(one(1, 2, 64).requires_grad_(), weight=dual(one(64))),
                 lambda: o.gated_norm_fwd(x, dual(x)), lambda: o.gated_norm_fwd(x, scale=dual(one(64))),
                 lambda: o.gated_norm_vjp(dual(x), None, x), lambda: o.gated_norm_vjp(None, dual(x), x), lambda: o.gated_norm_vjp(x, x, dual(x)),
                 lambda: o.gated_norm_vjp(x, x, x, x, gate=dual(one(64))),
                 lambda: o.quantize_rows(dual(x[0])), lambda: o.gemm_i8(a8, dual(one(2)), w8, one(5)), lambda: o.gemm_i8(a8, one(2), w8, one(5), dual(one(5))),
                 lambda: o.gemm_i8(a8, one(2), w8, one(5), epi="resid", resid=dual(one(2, 5))),
                 lambda: o.linear_i8(dual(x[0]), w8, one(5)), lambda: o.linear_i8(x[0], w8, dual(one(5))),
                 lambda: o.shared_prefix_attention(dual(q), k, k), lambda: o.shared_prefix_attention(q, dual(k), k),
                 lambda: o.shared_prefix_attention(q, k, dual(k)), lambda: o.shared_prefix_attention(q, k, k, dual(own), own),
                 lambda: o.shared_prefix_attention(q, k, k, own, dual(own))]
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for i, call in enumerate(calls):
                    with pytest.raises(err, match="forward-mode"):
                        call()
                        pytest.fail(f"call {i} was accepted")
        # tensors without a tangent are taken as outside the level
        r, h = o.gated_norm(x, x)
    for a, b in zip((r, h), o.gated_norm(x, x)):
        assert torch.equal(a, b)
    # a tangent that only the incoming gradient carries
    leaf = torch.randn(1, 2, 64, device="cuda", requires_grad=True)
    r, _ = o.gated_norm(leaf)
    with forward_ad.dual_level(), pytest.raises(err, match="forward-mode"):
        torch.autograd.grad(r, leaf, forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
@pytest.mark.parametrize("n,grp,p,more", [(5, 2, 0, 0), (40, 1, 0, 0), (40, 4, 0, 3), (150, 1, 0, 0), (150, 2, 0, 70), (90, 1, 100, 0), (64, 1, 64, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_infinite_value_stays_one(n, grp, p, more, dtype):
    """One infinite value among causal own keys is the result of every row that sees its key, with its sign, whatever tile it lies in; rows
    that do not see it keep their bits.  (Scores of normal draws over 64 dims: no weight is near the smallest 16-bit one.)"""
    q, pk, pv, ok, ov, _ = attention_case(2, n, 2 * grp, 2, 64, p, n + more, dtype, seed=n + p)
    want = ops().shared_prefix_attention(q, pk, pv, ok, ov)
    for at in sorted({0, 1, 31, 33, 45, 70, more, n // 2, n + more - 1} & set(range(n + more))):
        for bad in (math.inf, -math.inf, math.nan):
            v2 = ov.clone()
            v2[1, at, 1, 3] = bad
            got = ops().shared_prefix_attention(q, pk, pv, ok, v2)
            first = max(0, at - more)                                    # the first query that sees key `at`
            assert torch.equal(got[0], want[0]) and torch.equal(got[1, :first], want[1, :first]) and torch.equal(got[1, :, :grp], want[1, :, :grp]), (at, bad)
            there = got[1, first:, grp:, 3].float()
            assert (torch.isnan(there) if bad != bad else there == bad).all(), (at, bad)
            assert torch.isfinite(got[1, first:, grp:, [d for d in range(64) if d != 3]]).all(), (at, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8, 100])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_infinite_value_where_the_maximum_leaps(n, dtype):
    """Prefix keys whose weights vanish beside the own ones: what was summed before is multiplied by zero, an infinity of the new keys is not."""
    q, pk, pv, ok, ov, _ = attention_case(1, n, 1, 1, 64, 64, n, dtype, seed=n)
    q.zero_(), pk.zero_(), ok.zero_()
    q[..., 0], pk[..., 0] = 1, -200
    ov[0, n // 2, 0, 5] = -math.inf
    out = ops().shared_prefix_attention(q, pk, pv, ok, ov, scale=1.0)[0, :, 0]
    assert torch.isfinite(out[: n // 2]).all() and (out[n // 2:, 5] == -math.inf).all() and torch.isfinite(out[:, [d for d in range(64) if d != 5]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 0, 130), (3, 1, 4, 2, 700, 40), (1, 70, 2, 1, 100, 70), (2, 90, 1, 1, 0, 90)], ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype,top", [("f16", 60000.0), ("f16", 5000.0), ("f16", 900.0), ("bf16", 1e5), ("bf16", 1e15)])
def test_attention_scores_of_any_finite_size(case, dtype, top):
    """Scores far beyond what fp32 tells apart by one: a row's largest key alone remains, for finite q and k of any size.  q and k are
    whole multiples of powers of two, the same in all dims, the products exact; the runner-up lies 1 / 64 of the largest score below it."""
    b, n, h, hk, p, o = case
    q, pk, pv, ok, ov, _ = attention_case(b, n, h, hk, 64, p, o, dtype, seed=7)
    q.fill_(2.0 ** math.floor(math.log2(top)))
    k = [t for t in (pk, ok) if t is not None]
    g = torch.Generator().manual_seed(int(top))
    for t in k:
        t.copy_((torch.randint(-63, 64, (*t.shape[:-1], 1), generator=g) * 2.0 ** (math.floor(math.log2(top)) - 6)).to(t.dtype))
    out, lse = ops().shared_prefix_attention(q, pk, pv, ok, ov, return_lse=True)
    f = lambda t: t.double().cpu()  # noqa: E731
    for i in range(b):
        for t in range(n):
            seen = o - n + t + 1
            for j in range(h):
                kk = torch.cat(([f(pk[:, j // (h // hk), 0])] if p else []) + [f(ok[i, :seen, j // (h // hk), 0])])
                vv = torch.cat(([f(pv[:, j // (h // hk)])] if p else []) + [f(ov[i, :seen, j // (h // hk)])])
                s = kk * float(q[i, t, j, 0]) * 8                        # 64 dims over their root
                w = torch.softmax(s, 0)                              # ties share: at most 2 rounding steps of p and of the output
                want = w @ vv
                tol = 2 * half_step(q.dtype) * (w @ vv.abs()) + rounding(q.dtype, want)
                assert ((f(out[i, t, j]) - want).abs() <= tol).all(), (i, t, j)
                assert abs(float(lse[i, j, t]) - float(torch.logsumexp(s, 0))) <= 4 * E * float(s.abs().max()), (i, t, j)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(1, 1, 0, 640), (3, 2, 1280, 64), (1, 70, 640, 0), (2, 100, 0, 256)], ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("less", [25.1, 28.3])
def test_attention_tail_of_small_weights(case, dtype, less):
    """One key in 32 has a score above the others' by `less` in base-2 logarithms and values of zero, so that the result is the others'
    weights alone.  A weight is off by half a step of its type (bf16) or by 2^-32 of the largest (f16, whose smaller steps end there)."""
    b, n, p, o = case
    q, pk, pv, ok, ov, _ = attention_case(b, n, 2, 1, 64, p, o, dtype, seed=3)
    q.zero_()
    q[..., 0] = 1
    high = torch.tensor(less).to(q.dtype)
    for k, v in ((pk, pv), (ok, ov)):
        if k is None:
            continue
        axis = k.dim() - 3
        head = (torch.arange(k.shape[axis]) % 32 == 0).cuda().view(-1, 1, 1)
        k.zero_()
        k[..., 0] = torch.where(head, high.cuda(), torch.zeros((), dtype=q.dtype, device="cuda"))[..., 0]
        v.copy_(torch.where(head, torch.zeros((), dtype=q.dtype, device="cuda"), v.abs().clamp(0.5, 4) * (1024 if dtype == "f16" else 1)))
    out, lse = ops().shared_prefix_attention(q, pk, pv, ok, ov, causal=False, scale=math.log(2), return_lse=True)
    keys = torch.cat([t.double().cpu() for t in ([] if pk is None else [pk]) + ([] if ok is None else [ok[0]])])[:, 0, 0]
    for i in range(b):
        vals = torch.cat([t.double().cpu() for t in ([] if pv is None else [pv]) + ([] if ov is None else [ov[i]])])[:, 0]
        w = torch.softmax(keys * math.log(2), 0)
        want = w @ vals
        step = 2.0 ** -32 if dtype == "f16" else half_step(q.dtype) * 2.0 ** -float(high)
        tol = step * w.max() * vals.sum(0) + 64 * E * want + rounding(q.dtype, want)
        assert ((out[i].double().cpu() - want).abs() <= tol).all(), ((out[i].double().cpu() - want).abs() / tol).max()
        assert (lse[i].double().cpu() - torch.logsumexp(keys * math.log(2), 0)).abs().max() <= 64 * E * less


@pytest.mark.gpu
def test_contiguous_tensors_at_any_address():
    """Tensors that are contiguous but off the kernels' 16 bytes, or whose rows stand too far apart for them, are copied, not refused."""
    o = ops()
    g = torch.Generator().manual_seed(11)

    def off(t, by=1):
        """The same values, contiguous, `by` elements behind an allocation's start."""
        room = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
        room[by:].copy_(t.reshape(-1))
        moved = room[by:].view(t.shape)
        assert moved.is_contiguous() and moved.data_ptr() % 16
        return moved
    for d, n, b in ((64, 3, 2), (128, 40, 1)):
        q, pk, pv, ok, ov, lens = attention_case(b, n, 4, 2, d, 70, 50, "bf16", seed=d)
        names = dict(q=q, pk=pk, pv=pv, ok=ok, ov=ov)
        want = o.shared_prefix_attention(q, pk, pv, ok, ov, lens)
        for which in (["q"], ["pk"], ["pv"], ["ok"], ["ov"], list(names)):
            args = {k: off(v, 1 + 2 * i) if k in which else v for i, (k, v) in enumerate(names.items())}
            assert torch.equal(o.shared_prefix_attention(args["q"], args["pk"], args["pv"], args["ok"], args["ov"], lens), want), which
    a = torch.randint(-127, 128, (40, 256), generator=g, dtype=torch.int8).cuda()
    w = torch.randint(-127, 128, (30, 256), generator=g, dtype=torch.int8).cuda()
    sa, sw, x = torch.rand(40, generator=g).cuda(), torch.rand(30, generator=g).cuda(), torch.randn(40, 256, generator=g).cuda()
    want, layer = o.gemm_i8(a, sa, w, sw), o.linear_i8(x, w, sw)
    assert torch.equal(o.gemm_i8(off(a), off(sa), w, off(sw)), want) and torch.equal(o.gemm_i8(a, sa, off(w, 4), sw), want)
    assert torch.equal(o.gemm_i8(off(a[:1], 3), sa[:1], off(w[:1]), sw[:1]), want[:1, :1])
    assert torch.equal(o.linear_i8(off(x), off(w, 5), sw), layer) and torch.equal(o.linear_i8(off(x, 3)[:7], off(w, 5), off(sw)), o.linear_i8(x[:7], w, sw))
    # rows more than 2^22 bytes apart
    far = torch.empty(39 * ((1 << 22) + 16) + 256, dtype=torch.int8, device="cuda").as_strided((40, 256), ((1 << 22) + 16, 1))
    far.copy_(a)
    assert torch.equal(o.gemm_i8(far, sa, w, sw), want)
    far[:30].copy_(w)
    assert torch.equal(o.gemm_i8(a, sa, far[:30], sw), want) and torch.equal(o.linear_i8(x, far[:30], sw), layer)


@pytest.mark.gpu
@pytest.mark.parametrize("parts", ["gate scale shift", "scale", "shift", "scale shift", "gate shift"])
@pytest.mark.parametrize("case", [(256, 1, 7, "f32", "f32", "rms", "layer", True), (700, 3, 40, "bf16", "bf16", "layer", "rms", True), (300, 32, 512, "f16", "f32", "none", "layer", False),
                                  (1500, 2, 515, "bf16", "f32", "layer", "layer", True), (290, 5, 2048, "f16", "f16", "rms", "rms", True),
                                  (2300, 1, 1025, "f32", "f32", "layer", "layer", True), (257, 2, 8200, "bf16", "bf16", "rms", "layer", True)],
                         ids=lambda c: "-".join(map(str, c)))
def test_gated_norm_many_short_samples_with_parameters_of_their_own(case, parts):
    """Gradients of scale, shift and gate where a team of lanes takes whole samples, and of what all samples share beside them."""
    b, s, d, dtype, params, post, pre, affine = case
    t, kw, (gr, gh) = norm_case(b, s, d, dtype, params, post, pre, "sample" if "gate" in parts else "none", False, affine, seed=b)
    g = torch.Generator().manual_seed(s)
    for n in ("scale", "shift"):
        if n in parts:
            kw[n] = torch.randn(b, d, generator=g).mul(.3).to(torch.float32 if params == "f32" else t["x"].dtype).cuda()
    val, tol = norm64(t["x"], t["y"], **kw, grad_r=gr, grad_h=gh)
    got = ops().gated_norm_vjp(gr, gh, t["x"], t["y"], **kw)
    for n, v in got.items():
        if v is not None:
            within(v, val["g_" + n], tol["g_" + n] + rounding(v.dtype, val["g_" + n]), n)
    assert sorted(n for n in got if got[n] is not None) == sorted(n[2:] for n in val if n.startswith("g_"))
    # every gradient for itself: the same bits
    for n in [n for n in got if got[n] is not None]:
        assert torch.equal(ops().gated_norm_vjp(gr, gh, t["x"], t["y"], **kw, wanted=(n,))[n], got[n]), n


def test_attention_requests_do_not_read_a_descriptor_just_written(tmp_path):
    """The requests to LDS are written in assembly, where the compiler does not see what they read: a descriptor or an address in scalar
    registers that a vector instruction (a restored spill, for one) wrote needs five wait states, and M0 has no other user."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    out = tmp_path / "attention.s"
    run = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fno-gpu-rdc", "-w", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                          "--cuda-device-only", "-S", "-I", str(REPO / PKG / "csrc"), str(REPO / PKG / "csrc" / "prefix_attention.hip"), "-o", str(out)],
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-1500:]

    def scalars(text):
        regs = set()
        for a, b, c in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
            regs |= {int(c)} if c else set(range(int(a), int(b) + 1))
        return regs
    behind, in_asm, requests = [], False, 0                 # (scalar registers that a vector instruction wrote, its wait states), newest last
    for raw in out.read_text().split("\n"):
        line = raw.strip()
        if line.startswith((";;#ASMSTART", ";;#ASMEND")):
            in_asm = line.startswith(";;#ASMSTART")
            continue
        code = line.split(";")[0].strip()
        if not code or code.startswith("."):
            continue
        if code.endswith(":"):                              # (what ran before a label is taken to be what stands before it)
            continue
        assert in_asm or not re.search(r"\bm0\b", code), code
        if code.startswith("buffer_"):
            requests += in_asm
            states = 0
            for regs, n in reversed(behind):
                if states >= 5:
                    break
                assert not regs & scalars(code), code
                states += n
        nop = re.match(r"s_nop (\w+)", code)
        behind.append((scalars(code.split(None, 1)[1].split(",")[0]) if code.startswith("v_") and " " in code else set(), int(nop[1], 0) + 1 if nop else 1))
        behind = behind[-8:]
    assert requests >= 8 * 12
