"""Calls of the operators of strassen_hip/block.py that are easy to get wrong around their kernels: together with the other features of
the framework, on memory that is shared, under torch's transforms and hooks.  What needs no GPU runs without one."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import block_reference as ref


def _randn(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


# ------------------------------------------------------------------------------------------ the swap of Linear layers
def test_swap_of_linear_layers_keeps_epilogues():
    """A LinearAct has an activation and takes a residual, which no Strassen layer has: it stays what it is."""
    from model.layers import LinearAct, LinearStrassen, LinearStrassenRect, replace_linear_with_strassen
    import torch.nn as nn
    layers = lambda: nn.ModuleDict({"act": LinearAct(256, 256, activation="silu", device="cpu"), "wide": LinearAct(256, 512, activation="gelu", device="cpu"),
                                    "plain": LinearAct(256, 256, device="cpu"), "inner": nn.Sequential(LinearAct(128, 128, activation="relu", device="cpu"), nn.Linear(128, 128))})
    for square_only in (True, False):
        m = layers()
        acts = [m["act"], m["wide"], m["plain"], m["inner"][0]]
        replace_linear_with_strassen(m, square_only=square_only)
        assert [m["act"], m["wide"], m["plain"], m["inner"][0]] == acts
        assert type(m["inner"][1]) is (LinearStrassen if square_only else LinearStrassenRect)


@pytest.mark.gpu
def test_fused_block_after_the_swap():
    """gpt_block_demo's FusedBlock gives the same bits before and after the swap of its Linear layers."""
    import gpt_block_demo as demo
    from model.layers import replace_linear_with_strassen
    torch.manual_seed(0)
    for square_only in (True, False):
        block = demo.FusedBlock(demo.Block(256, 4, dtype=torch.bfloat16, rotary=True))
        x = _randn((2, 70, 256), torch.bfloat16, 1).cuda()
        with torch.no_grad():
            before = block(x)
            replace_linear_with_strassen(block, square_only=square_only)
            assert torch.equal(block(x), before)


# ------------------------------------------------------------------------------------- rotary on memory that is shared
def _packed(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _pairs():
    """(q, k, whether they have an element in common)"""
    t, h, p, a = _packed(2, 9, 8, 16), _packed(2, 9, 4, 3, 16), _packed(2, 9, 8, 16), _packed(3, 10, 6, 16)
    return [
        (t[:, :, :4], t[:, :, 4:6], False), (t[:, :, :4], t[:, :, 3:6], True), (t[:, :, ::2], t[:, :, 1::2], False), (t[:, :, ::2], t[:, :, 2::4], True),
        (t[:, :-1], t[:, 1:], True), (t[:, :4], t[:, 4:], False), (t[:, :5], t[:, 4:], True), (t[:1], t[1:], False), (t, t, True),
        (h[:, :, :, 0], h[:, :, :, 1], False), (h[:, :, :, 1], h[:, :, :, 0], False), (h[:, :, :, 0], h[:, :, 2:, 0], True), (h[:, :, :2, 2], h[:, :, 1:, 2], True),
        (p[:, :, :4], p[:, :, 3:8:2], True), (p[:, :, :4], p[:, :, 4:8:2], False), (p[:, :, 1:8:2], p[:, :, ::4], False), (p[:, ::2], p[:, 1::2][:, :, ::2], False),
        (p[..., :8], p[..., 8:], False), (p[..., :9], p[..., 8:], True), (t, p, False), (a.transpose(1, 2)[:, :2], a.transpose(1, 2)[:, 2:], False),
        (a[:, ::3], a[:, 1::3], False), (a[:, ::3], a[:, ::2], True), (a[:, 1::4], a[:, ::2], False), (a[:, :0], a, False),
        (t[:, :1].expand(2, 9, 8, 16), t[:, 1:], False), (t[:, :1].expand(2, 9, 8, 16), t[:, :2], True),
    ]


def _bytes(t):
    """Every byte of a tensor's elements."""
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    es = t.element_size()
    return set((t.data_ptr() + es * at.flatten()[:, None] + torch.arange(es)).flatten().tolist())


def test_memory_in_common():
    from strassen_hip.block import _ext
    share = _ext().share
    for i, (q, k, want) in enumerate(_pairs()):
        assert bool(_bytes(q) & _bytes(k)) == want, i   # the table itself
        assert share(q, k) == want and share(k, q) == want, i


def test_memory_in_common_of_any_strides():
    """Small random strides and places, elements of two and four bytes that may begin inside one another."""
    import random
    from strassen_hip.block import _ext
    share, overlaps_itself = _ext().share, _ext().overlaps_itself
    rng, seen = random.Random(5), [0, 0, 0, 0]
    raw = bytearray(4096)
    for _ in range(3000):
        dtype = rng.choice((torch.bfloat16, torch.float32))
        views = []
        for _ in range(2):
            base = torch.frombuffer(raw, dtype=dtype, count=1024 - 2, offset=rng.choice((0, 0, 0, 1, 2)))
            views.append(torch.as_strided(base, [rng.randint(1, 4) for _ in range(4)], [rng.choice((1, 2, 3, 5, 8, 12, 31, 60)) for _ in range(4)], rng.randint(0, 300)))
        q, k = views
        want = bool(_bytes(q) & _bytes(k))
        assert share(q, k) == want, (q.shape, q.stride(), k.shape, k.stride())
        itself = len(_bytes(q)) < q.numel() * q.element_size()
        assert overlaps_itself(q) == itself, (q.shape, q.stride())
        seen[want] += 1
        seen[2 + itself] += 1
    assert min(seen) > 200


def test_memory_in_common_of_long_tensors_is_quick():
    """Strides that do not nest in one another: an answer after a bounded number of steps, yes where they run out."""
    import time
    from strassen_hip.block import _ext
    t = torch.zeros(8, 4096, 6, 16, dtype=torch.bfloat16)
    start = time.perf_counter()
    assert not _ext().share(t[:, :, :4], t[:, :, 4:]) and not _ext().share(t[:, ::2], t[:, 1::2])
    assert _ext().share(t[:, ::5], t[:, 4095 // 3::7])
    odd = torch.zeros(1 << 22, dtype=torch.bfloat16)
    _ext().share(torch.as_strided(odd, (97, 101, 103), (9973, 9967, 7)), torch.as_strided(odd, (89, 83, 79), (9949, 9941, 11), 3))
    assert time.perf_counter() - start < 1.0


@pytest.mark.gpu
def test_rotary_in_place_on_views():
    """What has no element in common turns in place, whatever its strides; the rest is refused and left as it was."""
    import strassen_hip as hip
    f, _ = hip.rotary_frequencies(8)
    for i, (q, k, common) in enumerate(_pairs()):
        if q.shape[:2] != k.shape[:2] or q.shape[-1] != k.shape[-1]:
            continue
        size = lambda t: 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0
        low = min(q.data_ptr(), k.data_ptr())
        whole = (max(q.data_ptr() + 2 * size(q), k.data_ptr() + 2 * size(k)) - low) // 2
        if whole > 1 << 20:   # two tensors
            continue
        buf = _randn((whole,), torch.bfloat16, i).cuda()
        gq, gk = (torch.as_strided(buf, t.shape, t.stride(), (t.data_ptr() - low) // 2) for t in (q, k))
        before, (wq, wk) = buf.clone(), hip.rotary(gq, gk, f)
        if common or 0 in gq.stride():
            with pytest.raises(ValueError, match="share memory"):
                hip.rotary(gq, gk, f, inplace=True)
            assert torch.equal(buf, before)
            continue
        hip.rotary(gq, gk, f, inplace=True)
        assert torch.equal(gq, wq) and torch.equal(gk, wk), i
        rest = torch.ones_like(buf, dtype=torch.bool)
        for t in (q, k):
            torch.as_strided(rest, t.shape, t.stride(), (t.data_ptr() - low) // 2).fill_(False)
        assert torch.equal(buf[rest], before[rest]), i


# -------------------------------------------------------------------------------------------------- hooks of autograd
def _operators(hip, seed=1):
    """name: (call, leaves): each operator on operands that are views with strides of their own."""
    wide = lambda shape, pad, s: _randn((*shape[:-1], shape[-1] + pad), torch.float32, seed + s).cuda()[..., :shape[-1]].detach().requires_grad_()
    f, _ = hip.rotary_frequencies(8)
    x, w, b, r, n = wide((5, 24), 3, 1), wide((40, 24), 5, 2), wide((40,), 0, 3), wide((5, 40), 4, 4), wide((24,), 0, 5)
    q, k = wide((2, 7, 3, 16), 2, 6), wide((2, 7, 1, 16), 4, 7)
    pos = torch.randint(0, 1000, (2, 70), generator=torch.Generator().manual_seed(seed)).cuda()[:, 3:66:9]   # (2, 7), strides 70 and 9
    return {"linear_act": (lambda: hip.linear_act(x, w, b, activation="gelu", residual=r), [x, w, b, r]), "layer_norm": (lambda: hip.layer_norm(x, n, n), [x, n]),
            "rotary": (lambda: torch.cat(hip.rotary(q, k, f, pos), 2), [q, k])}


def _turned(t):
    """The same values, the first dimension's elements side by side."""
    return t.transpose(0, -1).contiguous().transpose(0, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear_act", "layer_norm", "rotary"])
def test_saved_tensors_come_back_otherwise(name):
    """Hooks on saved tensors: to host memory and back, in another order, by checkpoints that compute them again.  What does not come back is said."""
    import strassen_hip as hip
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    from torch.utils.checkpoint import checkpoint
    call, leaves = _operators(hip)[name]
    y = call()
    dy = _randn(tuple(y.shape), torch.float32, 9).cuda()
    want = torch.autograd.grad(y, leaves, dy)
    keep = lambda t: t
    for hooks in (save_on_cpu(), saved_tensors_hooks(keep, _turned), saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda())):
        with hooks:
            y = call()
        for got, ref_ in zip(torch.autograd.grad(y, leaves, dy), want):
            assert torch.equal(got, ref_)
    for got, ref_ in zip(torch.autograd.grad(checkpoint(lambda _: call(), leaves[0], use_reentrant=False), leaves, dy), want):
        assert torch.equal(got, ref_)
    with saved_tensors_hooks(keep, lambda t: torch._neg_view(-t) if t.dtype.is_floating_point else t):
        y = call()
    for got, ref_ in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(got, ref_)
    with saved_tensors_hooks(keep, _Counted):
        y = call()
    with pytest.raises(RuntimeError):   # the subclass's own refusal of an operation, or "plain tensors"
        torch.autograd.grad(y, leaves, dy)
    for spoil in (lambda t: t.cpu(), lambda t: t[..., :1] if t.shape[-1] > 1 else t, lambda t: t.float() if t.dtype == torch.float64 else t.double()):
        with saved_tensors_hooks(keep, spoil):
            y = call()
        with pytest.raises(RuntimeError, match="came back as"):
            torch.autograd.grad(y, leaves, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear_act", "layer_norm", "rotary"])
def test_gradients_in_another_order(name):
    """A hook on the result gives its gradient other strides, or one value for all of it."""
    import strassen_hip as hip
    call, leaves = _operators(hip)[name]
    y = call()
    dy = _randn(tuple(y.shape), torch.float32, 9).cuda()
    want = torch.autograd.grad(y, leaves, dy)
    y = call()
    y.register_hook(_turned)
    for got, ref_ in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(got, ref_)
    one = torch.full((), 0.5).cuda()
    for got, ref_ in zip(torch.autograd.grad(call(), leaves, one.expand(y.shape)), torch.autograd.grad(call(), leaves, one.expand(y.shape).contiguous())):
        assert torch.equal(got, ref_)


# ------------------------------------------------------------------------------- forward mode, transforms, recorded programs
def _entries(hip, device):
    """Each entry point as a function of one tensor (4, 8)."""
    w, f = torch.ones(8, 8, device=device), torch.ones(2, dtype=torch.float64, device=device)
    return [lambda x: hip.linear_act(x, w), lambda x: hip.linear_act(w, x), lambda x: hip.linear_act(w, w, x[0]), lambda x: hip.linear_act(w[:4], w, residual=x),
            lambda x: hip.layer_norm(x), lambda x: hip.layer_norm(w, x[0]), lambda x: hip.layer_norm(w, None, x[0]),
            lambda x: hip.rotary(x.view(1, 2, 2, 8), None, f), lambda x: hip.rotary(w.view(1, 2, 4, 8), x.view(1, 2, 2, 8), f)[1], lambda x: hip.matmul(x, w), lambda x: hip.matmul(w[:, :4], x)]


@pytest.mark.parametrize("i", range(11))
def test_forward_mode_and_traces_are_refused(i):
    """Refused before anything else is looked at: no GPU is needed to see it."""
    import strassen_hip as hip
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    entry = _entries(hip, "cpu")[i]
    x = _randn((4, 8), torch.float32, 1)
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no forward-mode"):
            entry(dual)
        if i < 9:   # as in torch's own operations, there is no tangent where they are switched off
            with torch.inference_mode(), pytest.raises(RuntimeError, match="no CPU implementation"):
                entry(dual)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(entry, (x,), check_trace=False)
    if i < 9:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(entry)(x)
        with pytest.raises(RuntimeError, match="no torch.func|no forward-mode"):
            torch.func.jvp(entry, (x,), (x,))
        with pytest.raises(RuntimeError, match="no torch.func"):
            torch.func.vmap(lambda u: entry(u))(x[None])
        with pytest.raises(RuntimeError, match="no torch.func"):
            torch.func.grad(lambda u: entry(u).sum())(x)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        entry(x)


@pytest.mark.gpu
def test_forward_mode_over_gradients_is_refused():
    import strassen_hip as hip
    import torch.autograd.forward_ad as forward_ad
    for name, (call, leaves) in _operators(hip).items():
        y = call()
        dy = torch.ones_like(y)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode"):
            torch.autograd.grad(y, leaves, forward_ad.make_dual(dy, dy))
    for entry in _entries(hip, "cuda"):
        x = _randn((4, 8), torch.float32, 1).cuda()
        with forward_ad.dual_level():   # a level without a tangent changes nothing
            got = entry(x)
        assert torch.equal(got, entry(x))


# ------------------------------------------------------------------------------------------------------------- capture
@pytest.mark.gpu
def test_capture_looks_behind_views_and_results():
    """Operands that were computed from a leaf of a living eager graph, or computed eagerly themselves.  Forward alone is captured; the
    refusal comes before a backward pass could run."""
    import strassen_hip as hip
    f, _ = hip.rotary_frequencies(8)
    p = torch.zeros(24, 8, device="cuda", requires_grad=True)
    x = torch.zeros(3, 8, device="cuda")
    calls = [lambda: hip.linear_act(x, p[:8]), lambda: hip.linear_act(p.view(3, 64)[:, :8], x), lambda: hip.linear_act(x, x, (p[0] * 2)[:3]), lambda: hip.linear_act(x, x, residual=p[:3, 5:]),
             lambda: hip.layer_norm(x, p[1]), lambda: hip.layer_norm(torch.relu(p).sum(0)), lambda: hip.rotary(p.view(1, 4, 6, 8)[:, :, :4], None, f),
             lambda: hip.rotary(x.view(1, 1, 3, 8), p[None, None, :2], f)[1]]
    for call in calls:
        alive = call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        torch.cuda.synchronize()
        del alive
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        g.replay()
        torch.cuda.synchronize()
        assert out.requires_grad
        del out
    eager = torch.relu(p[:3])   # no other graph of p is alive, but this operand's own way back is the default stream's
    with pytest.raises(RuntimeError, match="computed there"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            hip.linear_act(eager, x)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_captured_gradients_through_views():
    """A training step whose weights are parts of one packed leaf: captured, replayed four times with eager work between."""
    import strassen_hip as hip
    f, _ = hip.rotary_frequencies(8)
    packed = _randn((64, 32), torch.bfloat16, 1, 0.2).cuda().requires_grad_()
    x, dy = _randn((3, 5, 32), torch.bfloat16, 2).cuda(), _randn((3, 5, 32), torch.bfloat16, 3).cuda()

    def step():
        h = hip.layer_norm(x, packed[0], packed[1])
        q = hip.rotary(hip.linear_act(h, packed[:32]).view(3, 5, 4, 8), None, f).reshape(3, 5, 32)
        y = hip.linear_act(q, packed[32:], activation="silu", residual=h)
        return y.detach(), torch.autograd.grad(y, packed, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for turn in range(4):
        x.copy_(_randn((3, 5, 32), torch.bfloat16, 20 + turn).cuda())
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


# -------------------------------------------------------------------------------------------------- the largest sizes
@pytest.fixture(scope="module")
def cli(tmp_path_factory):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_model"))
    import hostbuild
    if hostbuild.clang() is None:
        pytest.skip("no clang to build the kernels for the host")
    return hostbuild.build_block(str(tmp_path_factory.mktemp("calls")), "plain")


def _launches(cli, tmp_path, lines):
    """What each call would launch: (status, [(grid x, y, z, block x)])."""
    import subprocess
    script = tmp_path / "script"
    script.write_text("\n".join(["dry"] + lines) + "\n")
    r = subprocess.run([cli, str(script)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    out = [line.split() for line in r.stdout.splitlines()]
    assert len(out) == len(lines)
    return [(int(o[0]), [tuple(int(v) for v in launch.split(",")) for launch in o[1:]]) for o in out]


M = (1 << 30) - 1
ODD = 4099   # a row stride that no 16-byte chunk fits
LARGE = [(M, 4, 1), (M, 4, 32), (1 << 29, 4, 33), (M, 8, 64), (M, 4, 127), ((1 << 29) - 31, 5, 17), (1, 4, M), (9, 8, M), (16, 3, 1 << 29), (17, 8, M), (40, 4, M), (1 << 20, 64, 1 << 16), (3, M, 2), (40, M, 1)]


@pytest.mark.parametrize("code", [0, 1, 2])
def test_no_launch_is_larger_than_the_hardware_takes(cli, tmp_path, code):
    """Sizes up to 2^30 - 1, as far as a card's memory holds their operands: less than 2^32 threads in each direction of every launch, and
    together no fewer workgroups than the sizes need."""
    lines = []
    for m, k, n in LARGE:
        for pad in (0, ODD):
            lines.append("linear @ @ @ @ @ @ %d %d %d %d %d %d %d %d 4" % (m, k, n, k + pad, k + pad, n + pad, n + pad, code))
            for dx, dw in (("@", "@"), ("@", "-"), ("-", "@")):
                lines.append("linear_backward @ @ @ @ %s %s @ %d %d %d %d %d %d %d 4" % (dx, dw, m, k, n, n + pad, k + pad, k + pad, code))
    norms = [(M, 1), (1 << 23, 16385), ((1 << 23) + 5, 20000), (1, M), (1, 1 << 29), (70, 1 << 29), (M, 64)]
    for rows, cols in norms:
        lines.append("norm @ @ @ @ @ @ %d %d %d %d %d %d 1e-5" % (rows, cols, cols, cols, code, code))
        lines.append("norm_backward @ @ @ @ @ @ @ @ %d %d %d %d %d %d %d" % (rows, cols, cols, cols, cols, code, code))
    lines.append("rotary @ @ @ @ 1 %d 1 1 8 8 16 16 8 16 16 8 16 16 8 16 16 8 @ @ 64 0 1 0 1.0 0 0 %d" % (M, code))
    got = _launches(cli, tmp_path, lines)
    for line, (rc, launches) in zip(lines, got):
        assert rc == 0 and launches, line
        for gx, gy, gz, bx in launches:
            assert gx * bx < 1 << 32 and gy < 1 << 16 and gz == 1 and bx <= 1024, (line, gx, gy, bx)
    tail = got[8 * len(LARGE):]
    for (rows, cols), (_, fwd), (_, bwd) in zip(norms, tail[::2], tail[1::2]):
        sums = [g for g in bwd if g[1] == 2 and g[3] == 256][-(-(-cols // (1 << 24))):]
        assert sum(g[0] for g in sums) == -(-cols // 32), (rows, cols)
        if cols > 16384:
            assert sum(g[0] for g in fwd) == rows and sum(g[0] for g in bwd if g[3] == 512) == rows, (rows, cols)


def test_sizes_that_no_launch_holds_are_refused_before_any(cli, tmp_path):
    """More tiles than a launch holds whichever tile is taken: nothing is launched, not the activation's gradient either."""
    n = 1 << 20
    got = _launches(cli, tmp_path, ["linear @ @ @ @ @ @ %d 8 %d 8 8 %d %d 1 4" % (n, n, n, n), "linear_backward @ @ @ @ @ - @ %d %d 8 8 %d %d 1 4" % (n, n, n, n),
                                    "linear_backward @ @ @ @ - @ @ 8 %d %d %d %d %d 1 4" % (n, n, n, n, n)])
    assert got == [(-1, [])] * 3


@pytest.mark.gpu
def test_norm_over_several_launches():
    """Long rows and long column sums go in pieces: what lies on both sides of a border is what it is alone."""
    import strassen_hip as hip
    rows, cols = (1 << 16) + 3, 16389
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1)).requires_grad_()
    w, b = (_randn((cols,), torch.float32, 2 + i).cuda() for i in range(2))
    y = hip.layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, y.detach())
    for at in (slice(0, 2), slice((1 << 16) - 2, rows)):
        want = ref.norm(x[at].detach().cpu(), w.cpu(), b.cpu(), 1e-5, torch.bfloat16, torch.float32, y[at].detach().cpu())
        ref.check(y[at].detach(), want["y"])
        ref.check(dx[at], want["dx"])
    del x, y, dx
    cols = (1 << 24) + 37
    x, dy = _randn((3, cols), torch.float32, 5), _randn((3, cols), torch.float32, 6)
    gw, gb = (torch.ones(cols, device="cuda", dtype=torch.float32).requires_grad_() for _ in range(2))
    hip.layer_norm(x.cuda(), gw, gb).backward(dy.cuda())
    want = ref.norm(x, torch.ones(cols), torch.ones(cols), 1e-5, torch.float32, torch.float32, dy)
    ref.check(gw.grad, want["dw"])
    ref.check(gb.grad, want["db"])


@pytest.mark.gpu
def test_more_rows_than_small_tiles_hold():
    """2^29 rows and one output, forward and gradients: as 32 x 32 tiles they would be 2^32 threads."""
    import strassen_hip as hip
    rows = (1 << 29) + 5
    x = torch.empty(rows, 4, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1)).requires_grad_()
    w = _randn((1, 4), torch.float32, 2).cuda().requires_grad_()
    y = hip.linear_act(x, w, activation="relu")
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones((), device="cuda").expand(rows, 1))
    for at in (slice(0, 40), slice((1 << 28) - 20, (1 << 28) + 20), slice(rows - 40, rows)):
        xs = x[at].detach().cpu()
        want = ref.linear(xs, w.detach().cpu(), None, None, "relu", torch.float32, torch.ones(40, 1))
        ref.check(y[at].detach(), want["y"])
        ref.check(dx[at], want["dx"])
    # dw: a sum of 2^29 products; with splits and k-steps in fp32, n steps of the sum of magnitudes at most, sqrt(n) of them in earnest
    want = sum((piece.detach() * (piece.detach() @ w.detach().t() > 0)).double().sum(0) for piece in x.split(1 << 26))
    size = sum(piece.detach().abs().double().sum(0) for piece in x.split(1 << 26))
    assert ((dw[0].double() - want).abs() <= 2.0 ** 15 * ref.STEP * size).all(), (dw, want)


# ------------------------------------------------------------------------------------------------------------ the C ABI
def test_rotary_in_place_with_other_strides_is_refused():
    import ctypes
    from strassen_hip import _capi
    lib = _capi.load()
    strides = lambda *v: (ctypes.c_int64 * 3)(*v)
    here, there = ctypes.c_void_p(4096), ctypes.c_void_p(1 << 20)
    call = lambda q, k, qo, ko, qs, ks, qos, kos, tokens=2: lib.sthip_rotary(q, k, qo, ko, 1, tokens, 2, 2, 8, 8, qs, ks, qos, kos, here, None, 0, 0, 0, 0, 1.0, 0, 0, 2, None)
    packed, dense = strides(64, 32, 8), strides(32, 16, 8)
    assert call(here, None, here, None, packed, None, dense, None) == -3 and b"same strides" in lib.sthip_last_error()
    assert call(here, there, ctypes.c_void_p(8192), there, packed, packed, dense, dense) == -3
    assert call(here, there, here, there, packed, packed, dense, dense, tokens=0) == 0


def test_the_library_is_built_without_torch(monkeypatch, capsys):
    """Callers of the C ABI need no torch, neither does its build; the objects themselves are not compiled again here."""
    import importlib.util
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("sthip_build", os.path.join(root, "strassen-triton_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    monkeypatch.setattr(build, "_compile", lambda unit, force: (unit[0], "cached"))
    monkeypatch.setattr(build, "_run_torch", lambda cmd, what: pytest.fail("the torch side was built"))
    monkeypatch.setitem(sys.modules, "torch", None)   # import torch raises ImportError
    assert build.build() == build.LIB
    assert "left out" in capsys.readouterr().out


# ------------------------------------------------------------------------------------------- infinities in the epilogue
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [3, 70])   # few rows; tiles
def test_activations_and_slopes_at_the_ends(dt, name, rows):
    """z of any size, infinities and NaN, by way of the bias: act(inf) = inf and slope 1, beyond the reach of exp on the other side 0
    and slope 0 (relu exactly; the others' zero times -inf is NaN as in their formulas), NaN stays NaN."""
    import strassen_hip as hip
    inf, nan, big = float("inf"), float("nan"), 6e4 if dt == torch.float16 else 1e30
    z = torch.tensor([inf, -inf, nan, big, -big, 120.0, -120.0, 0.0] * 9)
    x, w = torch.zeros(rows, 24, dtype=dt).cuda(), _randn((72, 24), dt, 1).cuda()
    b = z.to(dt).cuda().requires_grad_()
    y = hip.linear_act(x, w, b, activation=name)
    (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
    low = z if name == "none" else torch.where(z < 0, torch.zeros(()), z)
    if name not in ("none", "relu"):
        low = torch.where(z == -inf, torch.tensor(nan), low)
    slope = torch.ones(72) if name == "none" else torch.where(z == 0, torch.tensor(0.0 if name == "relu" else 0.5), (z > 0).float())
    if name != "none":
        slope = torch.where(z != z, z, slope)
    y, db = y.detach().float().cpu(), db.float().cpu()
    want = low.to(dt).float()
    assert torch.equal(y.isnan(), want.isnan().expand(rows, 72)) and torch.equal(y.nan_to_num(1.0, 2e38, -2e38), want.nan_to_num(1.0, 2e38, -2e38).expand(rows, 72))
    assert torch.equal(db.isnan(), slope.isnan()) and torch.equal(db.nan_to_num(7.0), (rows * slope).nan_to_num(7.0))   # sums of whole and half numbers: exact


# --------------------------------------------------------------------------------- tensors whose memory is not their value
class _Counted(torch.Tensor):
    """A tensor whose operations are its own; without memory."""
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError


@pytest.mark.parametrize("i", range(9))
def test_tensors_without_memory_are_refused(i):
    import strassen_hip as hip
    from torch._subclasses.fake_tensor import FakeTensorMode
    entry = _entries(hip, "cpu")[i]
    x = _randn((4, 8), torch.float32, 1)
    if i in (0, 1, 3, 4):   # the others take a part of x first, which is the subclass's own affair
        with pytest.raises(RuntimeError, match="plain tensors"):
            entry(_Counted(x))
        with pytest.raises(RuntimeError, match="plain tensors"):
            entry(x.to_sparse())
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match="cannot be traced"):
        entry(x)


@pytest.mark.gpu
def test_pending_negations():
    """The imaginary part of a conjugate is a view that is yet to be negated."""
    import strassen_hip as hip
    negative = lambda t: torch.complex(t, t).conj().imag
    f, _ = hip.rotary_frequencies(8)
    x, w, b, r = (_randn(s, torch.float32, i).cuda() for i, s in enumerate([(5, 1), (6, 1), (6,), (5, 6)]))
    q = _randn((1, 4, 2, 16), torch.float32, 9).cuda()
    same = lambda got, want: torch.equal(got, want)
    assert negative(x).is_neg() and same(hip.linear_act(negative(x), w, b), hip.linear_act(-x, w, b))
    assert same(hip.linear_act(x, negative(w), negative(b), residual=negative(r)), hip.linear_act(x, -w, -b, residual=-r))
    assert same(hip.layer_norm(negative(r), negative(b), b), hip.layer_norm(-r, -b, b))
    flat = torch._neg_view(q)
    assert flat.is_neg() and flat.is_contiguous() and same(hip.rotary(flat, None, f), hip.rotary(-q, None, f)) and same(hip.layer_norm(flat), hip.layer_norm(-q))
    with pytest.raises(ValueError, match="negation"):
        hip.rotary(flat, None, f, inplace=True)
    leaf = r.clone().requires_grad_()
    y = hip.layer_norm(leaf, b)
    assert same(torch.autograd.grad(y, leaf, torch._neg_view(r))[0], torch.autograd.grad(hip.layer_norm(leaf, b), leaf, -r)[0])


# ---------------------------------------------------------------------------------------- the borders of few rows' own way
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d_in,d_out", [(8, 200, 4112), (9, 200, 4096), (9, 200, 4097), (16, 136, 5120), (16, 2051, 4100), (17, 200, 4096)])
def test_few_rows_on_both_sides_of_their_borders(dt, rows, d_in, d_out):
    import strassen_hip as hip
    x, w, b, r = (_randn(s, dt, 30 + i, std) for i, (s, std) in enumerate([((rows, d_in), 1.0), ((d_out, d_in), d_in ** -0.5), ((d_out,), 1.0), ((rows, d_out), 1.0)]))
    y = hip.linear_act(x.cuda(), w.cuda(), b.cuda(), activation="silu", residual=r.cuda())
    ref.check(y, ref.linear(x, w, b, r, "silu", dt)["y"])
