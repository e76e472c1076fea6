"""qk_norm_rope on the GPU against its formula in 64 bits, forward and backward."""

import math

import pytest
import torch

from rotary_reference import frequencies, pair_size, turned

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
STEP32 = 2.0 ** -24


def reference(q, k, positions, inv_freq, weights, eps, interleaved, dy=None):
    """Per side: (y, pair sizes before the turn), or with dy also (dx, its error's scale, dw, its error's scale)."""
    sides = []
    for i, x in enumerate((q, k)):
        x, w = x.double(), weights[i]
        d = x.shape[-1]
        r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt() if w is not None else torch.ones_like(x[..., :1])
        n = x * r
        scaled = n if w is None else n * w.double()
        res = [turned(scaled, positions, inv_freq, interleaved), pair_size(scaled, inv_freq.numel(), interleaved)]
        if dy is not None:
            u = turned(dy[i].double(), positions, inv_freq, interleaved, back=True)
            size = pair_size(dy[i].double(), inv_freq.numel(), interleaved)   # (turning back keeps it)
            if w is None:
                res += [u, size, None, None]
            else:
                g = u * w.double()
                res += [r * (g - n * (g * n).mean(-1, keepdim=True)),
                        r * (size * w.double().abs() + n.abs() * (size * w.double().abs() * n.abs()).mean(-1, keepdim=True)),
                        (u * n).sum((0, 1)), (size * n.abs()).sum((0, 1))]
        sides.append(res)
    return sides


def check(got, want, scale, dtype, steps, what):
    """Half a step of the type, and `steps` roundings of 32 bits (2^-24 each) of numbers of size `scale`."""
    smallest = {BF16: 0.0, FP16: 2.0 ** -25, FP32: 0.0}[dtype]
    bound = torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + steps * STEP32 * scale + smallest + 1e-30
    off = (got.double() - want).abs()
    assert got.dtype == dtype and bool((off <= bound).all()), (what, (off / bound).max().item())


# An angle is off by at most 2^-24 of a turn and 2^-24 of its sine and cosine each: below 10 * 2^-24 of the pair; the norm's sum
# of up to 128 squares, root and products stay below D / 2 + 8 roundings.
def forward_steps(d):
    return 10 + d / 2 + 8


def make(tokens, heads, kv_heads, d, dtype, seed=0, far=0):
    g = torch.Generator().manual_seed(seed)
    q, k, dq, dk = (torch.randn((tokens, h, d), generator=g).to(dtype).cuda() for h in (heads, kv_heads, heads, kv_heads))
    positions = torch.randint(0, 4 * tokens + 1, (tokens,), generator=g).cuda() + far
    weights = [(1 + 0.3 * torch.randn(d, generator=g)).cuda() for _ in range(2)]
    return q * 3, k, dq, dk, positions, weights


CASES = [  # tokens, heads, kv heads, head_dim, rotated pairs, interleaved, dtype, weights' dtype or "", far
    (1, 32, 8, 128, 64, False, BF16, BF16, 1 << 20),
    (5, 4, 1, 128, 64, True, FP16, FP32, 0),
    (37, 5, 3, 128, 32, False, BF16, FP32, 1 << 30),
    (130, 8, 8, 64, 32, False, FP16, FP16, 0),
    (63, 7, 1, 64, 16, True, BF16, BF16, 100),
    (64, 3, 2, 96, 48, False, BF16, BF16, 0),
    (17, 2, 1, 96, 24, True, FP16, FP16, 0),
    (9, 6, 2, 8, 4, False, BF16, FP32, 0),
    (33, 1, 1, 24, 8, True, FP16, FP16, 0),
    (1000, 8, 2, 128, 64, False, BF16, "", 0),
    (301, 17, 1, 72, 36, False, FP16, "q", 0),
    (40, 3, 2, 64, 32, False, BF16, "k", 0),
    (5003, 8, 2, 128, 64, False, BF16, BF16, 0),
    (9000, 4, 4, 64, 32, True, FP16, FP32, 1 << 17),
]


def weights_of(weights, dtype, kind):
    if kind == "":
        return [None, None]
    if kind == "q":
        return [weights[0].to(dtype), None]
    if kind == "k":
        return [None, weights[1].to(dtype)]
    return [w.to(kind) for w in weights]


@pytest.mark.parametrize("tokens,heads,kv_heads,d,pairs,interleaved,dtype,kind,far", CASES)
def test_forward_and_backward(tokens, heads, kv_heads, d, pairs, interleaved, dtype, kind, far):
    from moba_amd import qk_norm_rope
    print("norm_rope", tokens, heads, kv_heads, d, pairs, interleaved, dtype, kind, far, flush=True)
    q, k, dq, dk, positions, weights = make(tokens, heads, kv_heads, d, dtype, far=far)
    inv_freq, weights, eps = frequencies(pairs, "cuda"), weights_of(weights, dtype, kind), 1e-5
    plain = qk_norm_rope(q, k, positions, inv_freq, *weights, eps=eps, interleaved=interleaved)
    leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, *weights)]
    y = qk_norm_rope(leaves[0], leaves[1], positions.int() if far < 1 << 30 else positions, inv_freq, *leaves[2:], eps=eps,
                     interleaved=interleaved)
    present = [x for x in leaves if x is not None]
    grads = iter(torch.autograd.grad(y, present, (dq, dk)))
    grads = [None if x is None else next(grads) for x in leaves]
    want = reference(q, k, positions, inv_freq, weights, eps, interleaved, (dq, dk))
    for i, side in enumerate("qk"):
        assert torch.equal(plain[i], y[i]) and y[i].is_contiguous()
        ref = want[i]
        check(y[i], ref[0], ref[1], dtype, forward_steps(d), "y " + side)
        check(grads[i], ref[2], ref[3], dtype, 3 * forward_steps(d), "d" + side)
        if weights[i] is not None:
            # a wave adds its rows one after the other, at most heads * ceil(tokens / 1024); then 64 / 8 rows and 4 waves
            serial = (heads if i == 0 else kv_heads) * -(-tokens // 1024) + 16
            check(grads[i + 2], ref[4], ref[5], weights[i].dtype, serial + forward_steps(d) + 10, "d weight " + side)


def test_gradients_against_differences():
    """The operator's gradient along a direction against the change of its plain form in 64 bits along that direction."""
    from moba_amd import qk_norm_rope
    q, k, dq, dk, positions, weights = make(50, 4, 2, 64, BF16, seed=3)
    inv_freq = frequencies(32, "cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, weights[0], weights[1])]
    grads = torch.autograd.grad(qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:]), leaves, (dq, dk))

    def value(q, k, a, b):
        sides = reference(q, k, positions, inv_freq, [a, b], 1e-6, False)
        return (sides[0][0] * dq.double()).sum() + (sides[1][0] * dk.double()).sum()

    g = torch.Generator(device="cuda").manual_seed(1)
    base = [x.detach().double() for x in leaves]
    for i, x in enumerate(base):
        way, h = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64), 1e-5
        ends = [value(*(b + s * h * way if j == i else b for j, b in enumerate(base))) for s in (1, -1)]
        change, along = (ends[0] - ends[1]).item() / (2 * h), (grads[i].double() * way).sum().item()
        # half a step of bf16 of every product, as independent errors, four of their deviations; and h^2
        spread = (grads[i].double() * way).norm().item() * (2.0 ** -8 if i < 2 else 2.0 ** -20)
        assert abs(change - along) <= 4 * spread + 1e-6 * abs(change) + 1e-6, (i, change, along, spread)


def test_views_and_broadcast_inputs():
    from moba_amd import qk_norm_rope
    g = torch.Generator(device="cuda").manual_seed(5)
    inv_freq, positions = frequencies(64, "cuda"), torch.arange(50, device="cuda")
    w = torch.rand(128, generator=g, device="cuda").to(BF16) + 0.5
    fused = torch.randn((50, 12, 128), generator=g, device="cuda").to(BF16)
    views = [(fused[:, :8], fused[:, 8:10]),                                              # slices of a fused projection
             (fused.transpose(0, 1).contiguous().transpose(0, 1)[:, :8], fused[:, 10:]),  # heads outside
             (fused[:, :8, ::1].flip(0), fused[:, 8:10]),
             (torch.randn((50, 8, 256), generator=g, device="cuda").to(BF16)[..., ::2], fused[:, 8:10]),   # copied
             (torch.randn(50 * 4 * 130 + 1, generator=g, device="cuda").to(BF16)[1:].view(50, 4, 130)[..., :128], fused[:, 8:9]),
             (fused[:, :1].expand(50, 6, 128), fused[:1, 8:10].expand(50, 2, 128))]
    for q, k in views:
        got = qk_norm_rope(q, k, positions, inv_freq, w, w)
        want = qk_norm_rope(q.contiguous(), k.contiguous(), positions, inv_freq, w, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a head shared by expansion gets the sum of its copies' gradients
    head = fused[:, :1].detach().requires_grad_()
    copies = fused[:, :1].expand(50, 6, 128).contiguous().requires_grad_()
    dy = torch.randn((50, 6, 128), generator=g, device="cuda").to(BF16)
    k = fused[:, 8:10]
    one, = torch.autograd.grad(qk_norm_rope(head.expand(50, 6, 128), k, positions, inv_freq, w, w)[0], head, dy)
    many, = torch.autograd.grad(qk_norm_rope(copies, k, positions, inv_freq, w, w)[0], copies, dy)
    want = many.double().sum(1, keepdim=True)
    # (torch adds the six copies in 32 bits and rounds once)
    assert bool(((one.double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + 6 * STEP32 * many.double().abs().sum(1, keepdim=True) + 1e-30).all())


def test_odd_inputs():
    from moba_amd import qk_norm_rope
    inv_freq, w = frequencies(64, "cuda"), torch.ones(128, device="cuda", dtype=BF16)
    # no tokens
    q, k = (torch.empty((0, h, 128), device="cuda", dtype=BF16, requires_grad=True) for h in (4, 2))
    ww = w.clone().requires_grad_()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    y = qk_norm_rope(q, k, none, inv_freq, ww, w)
    assert y[0].shape == (0, 4, 128) and y[1].shape == (0, 2, 128)
    grads = torch.autograd.grad(y, (q, k, ww), y)
    assert grads[0].shape == q.shape and not grads[2].any()
    # rows of zeros and rows that are not finite stay with themselves; negative positions turn the other way
    q = torch.randn((4, 4, 128), device="cuda").to(BF16)
    q[0, 1], q[1, 2, 5], q[2, 3, 70] = 0, float("nan"), float("inf")
    positions = torch.tensor([0, -7, 3, -1000000], device="cuda")
    k = torch.randn((4, 1, 128), device="cuda").to(BF16)
    y, yk = qk_norm_rope(q, k, positions, inv_freq, w, w)
    want = reference(q, k, positions, inv_freq, [w, w], 1e-6, False)
    assert not y[0, 1].any() and y[1, 2].isnan().all() and not y[2, 3].isfinite().all()
    fine = torch.ones((4, 4), dtype=torch.bool, device="cuda")
    fine[1, 2] = fine[2, 3] = False
    check(y[fine], want[0][0][fine], want[0][1][fine], BF16, forward_steps(128), "y")
    check(yk, want[1][0], want[1][1], BF16, forward_steps(128), "yk")
    # only one result asked for
    leaf = k.clone().requires_grad_()
    ww = w.clone().requires_grad_()
    y = qk_norm_rope(k, leaf, positions, inv_freq, ww, w)
    dk, dw = torch.autograd.grad(y[1].float().sum(), (leaf, ww))
    assert dk.isfinite().all() and not dw.any()


def test_elements_that_are_not_turned_stay_alone():
    """An infinity or a NaN among them reaches no other element, forward or backward."""
    from moba_amd import qk_norm_rope
    q, k, dq, dk, positions, _ = make(6, 2, 1, 96, BF16)
    inv_freq = frequencies(24, "cuda")
    q[:, 0, 60], q[:, 1, 90], dq[:, 0, 70], dk[:, 0, 64] = float("inf"), float("nan"), float("-inf"), float("nan")
    leaf, leaf_k = q.clone().requires_grad_(), k.clone().requires_grad_()
    for interleaved in (False, True):
        y = qk_norm_rope(leaf, leaf_k, positions, inv_freq, interleaved=interleaved)
        g = torch.autograd.grad(y, (leaf, leaf_k), (dq, dk))
        for got, given in ((y[0], q), (y[1], k), (g[0], dq), (g[1], dk)):
            assert torch.equal(got[..., 48:].isfinite(), given[..., 48:].isfinite()) and got[..., :48].isfinite().all()
            fine = given[..., 48:].isfinite()
            assert torch.equal(got[..., 48:][fine], given[..., 48:][fine])


def test_same_bits_every_time_on_every_stream_and_in_a_graph():
    from moba_amd import qk_norm_rope
    q, k, dq, dk, positions, weights = make(3000, 8, 2, 128, BF16, seed=7)
    inv_freq = frequencies(64, "cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, weights[0], weights[1])]

    def both():
        y = qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:])
        return [*(v.detach() for v in y), *torch.autograd.grad(y, leaves, (dq, dk))]

    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = both()
    for _ in range(3):
        for x in static:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, want))
        assert all(torch.equal(a, b) for a, b in zip(both(), want))


@pytest.mark.parametrize("native", [True, False])
def test_a_capture_beside_a_living_graph_of_the_same_leaves_is_refused(native, monkeypatch):
    """Its backward pass would join the captured stream to the one that the leaves' gradients belong to.  No backward pass runs
    before the eager graph has gone."""
    from moba_amd import _lib, qk_norm_rope
    q, k, dq, dk, positions, weights = make(20, 4, 2, 64, BF16, seed=5)
    inv_freq, leaves = frequencies(32, "cuda"), [x.detach().requires_grad_() for x in (q, k, *weights)]
    if not native:
        monkeypatch.setattr(_lib.host(), "norm_rope", lambda *a: NotImplemented)
    alive = qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:])
    want = [y.detach().clone() for y in alive]
    torch.cuda.synchronize()
    graph, held = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    for a, b in (((leaves[0], k), ()), ((q, leaves[1]), weights), ((q, k), (leaves[2], weights[1])), ((q, k), (None, leaves[3]))):
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                held.add_(1)
                qk_norm_rope(*a, positions, inv_freq, *b)
    with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():   # (no backward pass: not refused)
        qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:])
    del alive
    with torch.cuda.graph(graph):
        y = qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:])
        g = torch.autograd.grad(y, leaves, (dq, dk))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(y, want)) and all(x.isfinite().all() for x in g)


def test_before_the_attention():
    """Training as it is used: norm and rotation, the packed attention behind them, one backward through both."""
    from moba_amd import moba_attn_varlen_gqa, qk_norm_rope
    from oracle import moba_oracle as O
    cu = [0, 300, 650]
    g = torch.Generator().manual_seed(11)
    q, k, v, do = (torch.randn((650, h, 128), generator=g).to(BF16).cuda() for h in (4, 2, 2, 4))
    positions = torch.cat([torch.arange(300), torch.arange(350)]).cuda()
    w = [(1 + 0.2 * torch.randn(128, generator=g)).to(BF16).cuda() for _ in range(2)]
    inv_freq, cu_t = frequencies(64, "cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, v, *w)]
    yq, yk = qk_norm_rope(leaves[0], leaves[1], positions, inv_freq, leaves[3], leaves[4])
    out = moba_attn_varlen_gqa(yq, yk, leaves[2], cu_t, 350, 1024, 3)     # one chunk a sequence: plain causal attention
    grads = torch.autograd.grad(out, leaves, do)
    # the same in 32 bits on the CPU, from the operator's rounded q and k on for the attention, exactly before
    yq32, yk32, v32 = (x.detach().float().cpu().requires_grad_() for x in (yq, yk, v))
    ref = O.moba_attn_varlen_oracle(yq32, yk32.repeat_interleave(2, 1), v32.repeat_interleave(2, 1), cu, 350, 1024, 3)
    ref.backward(do.float().cpu())
    # (the tolerances of the operator's own tests for its outputs and gradients)
    assert (out.detach().float().cpu() - ref.detach()).abs().max() < 2e-2
    assert (grads[2].float().cpu() - v32.grad).abs().max() < 4e-2
    want = reference(q, k, positions, inv_freq, w, 1e-6, False, (yq32.grad.cuda(), yk32.grad.cuda()))
    for i in range(2):
        off = (grads[i].double() - want[i][2]).norm() / want[i][2].norm()
        assert off < 2e-2, (i, off.item())
        off = (grads[3 + i].double() - want[i][4]).norm() / want[i][4].norm()
        assert off < 2e-2, (i, off.item())


def test_refusals_on_the_gpu():
    from moba_amd import qk_norm_rope
    q, k, _, _, positions, w = make(4, 2, 1, 64, BF16)
    f = frequencies(32, "cuda")
    with pytest.raises(ValueError, match="one device"):
        qk_norm_rope(q, k, positions.cpu(), f)
    with pytest.raises(ValueError, match="one device"):
        qk_norm_rope(q, k, positions, f, w[0].cpu())
    leaf = q.detach().requires_grad_()
    y, _ = qk_norm_rope(leaf, k, positions, f)
    g, = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)


def test_the_general_path_gives_the_same(monkeypatch):
    """The native call takes contiguous tensors and views alike; what it leaves to the Python path is computed the same."""
    from moba_amd import _lib, qk_norm_rope
    q, k, dq, dk, positions, weights = make(70, 6, 2, 128, FP16, seed=2)
    inv_freq, native = frequencies(32, "cuda"), _lib.host().norm_rope
    taken = []

    def both():
        leaves = [x.detach().requires_grad_() for x in (q, k, *weights)]
        y = qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:], interleaved=True)
        taken.append(type(y[0].grad_fn).__name__)
        return [*(v.detach() for v in y), *torch.autograd.grad(y, leaves, (dq, dk)), *qk_norm_rope(q, k, positions, inv_freq)]

    want = both()
    monkeypatch.setattr(_lib.host(), "norm_rope", lambda *a: NotImplemented)
    got = both()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and taken[0] != taken[1]
    monkeypatch.setattr(_lib.host(), "norm_rope", native)
    for args in ((q[:0], k[:0], positions[:0], inv_freq), (q, k.cpu(), positions, inv_freq), (q.float(), k, positions, inv_freq),
                 (q, k, positions[:5], inv_freq), (q, k, positions, inv_freq[:3]), (q, k, positions.view(1, -1), inv_freq)):
        assert native(*args, None, None, 1e-6, False) is NotImplemented
    with pytest.raises(TypeError):
        native(q, k)


def test_the_native_call_lets_other_threads_run():
    """In the entry point's place stands CPython's own PyGILState_Check, whose answer -- 1 with the lock -- would be an error code."""
    import ctypes
    from moba_amd import _lib, qk_norm_rope
    q, k, _, _, positions, _ = make(4, 2, 1, 64, BF16)
    try:
        _lib.bind_layer(_lib.host(), moba_qk_norm_rope=ctypes.pythonapi.PyGILState_Check)
        assert qk_norm_rope(q, k, positions, frequencies(32, "cuda"))[0].shape == q.shape
        _lib.bind_layer(_lib.host(), moba_qk_norm_rope=ctypes.pythonapi.Py_IsInitialized)     # (1: an error)
        with pytest.raises(RuntimeError, match="moba_qk_norm_rope failed with code 1"):
            qk_norm_rope(q, k, positions, frequencies(32, "cuda"))
    finally:
        _lib.bind_layer(_lib.host())


PI = 314159265358979323846264338327950288419716939937510582097494459230781640628620899  # * 10^-80


def exact_turn(position, inv_freq):
    """cos and sin of position * inv_freq, whose whole turns are taken off in whole numbers."""
    top, bottom = inv_freq.as_integer_ratio()
    top *= position
    turn = 2 * PI * bottom
    rest = (top * 10 ** 80) % turn                       # of an angle of rest / 10^80 / bottom
    if 2 * rest > turn:
        rest -= turn
    angle = rest / (10 ** 80 * bottom)                    # (a quotient of whole numbers, rounded once)
    return math.cos(angle), math.sin(angle)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_angles_of_far_positions(dtype):
    """Up to the last position that a double tells from the next, at frequencies of 1 and more as well."""
    from moba_amd import qk_norm_rope
    g = torch.Generator().manual_seed(2)
    positions = [s * (2 ** e + i) for e in (20, 30, 31, 34, 40, 45, 50, 52) for s, i in ((1, 0), (-1, 12345), (1, 777))] + [2 ** 53]
    inv_freq = torch.cat([frequencies(24), torch.tensor([1.0, 3.0, 1000.0, 0.7, 2.0 ** -30, 1e-20, 0.0, 123456.789])])
    x = torch.randn((len(positions), 2, 64), generator=g).to(dtype)
    x[:, 1, :32], x[:, 1, 32:] = 1, 0                     # (the angle's cosine and sine themselves)
    got, _ = qk_norm_rope(x.cuda(), x.cuda(), torch.tensor(positions).cuda(), inv_freq.cuda())
    cs = torch.tensor([[exact_turn(p, f) for f in inv_freq.tolist()] for p in positions], dtype=torch.float64)
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x.double()[..., :32], x.double()[..., 32:]
    want = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    check(got.cpu(), want, pair_size(x.double(), 32), dtype, forward_steps(0), "y")


@pytest.mark.parametrize("native", [True, False])
def test_derivatives_that_there_are_none_of(native, monkeypatch):
    import torch.autograd.forward_ad as fwd
    from moba_amd import _lib, qk_norm_rope
    q, k, dq, dk, positions, w = make(20, 4, 2, 64, BF16, seed=6)
    f = frequencies(32, "cuda")
    if not native:
        monkeypatch.setattr(_lib.host(), "norm_rope", lambda *a: NotImplemented)
    args, leaf = [q, k, positions, f, *w], q.clone().requires_grad_()
    want = qk_norm_rope(*args)
    y = qk_norm_rope(leaf, *args[1:])
    with fwd.dual_level():
        for i in (0, 1, 3, 4, 5):
            for where in (torch.enable_grad, torch.no_grad):
                with where(), pytest.raises(RuntimeError, match="forward-mode"):
                    qk_norm_rope(*[fwd.make_dual(x, torch.ones_like(x)) if i == j else x for j, x in enumerate(args)])
        for dy in ((fwd.make_dual(dq, dq), dk), (dq, fwd.make_dual(dk, dk))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(*args), want))
        assert torch.autograd.grad(y, leaf, (dq, dk))[0].isfinite().all()
    learned = f.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient of inv_freq"):
        qk_norm_rope(q, k, positions, learned)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(q, k, positions, learned, *w), want))


@pytest.mark.parametrize("native", [True, False])
def test_saved_tensors_that_come_back_otherwise(native, monkeypatch):
    """Hooks on saved tensors keep values, not strides and alignment."""
    from moba_amd import _lib, qk_norm_rope
    q, k, dq, dk, positions, weights = make(30, 4, 2, 64, BF16, seed=8)
    inv_freq = frequencies(32, "cuda")
    if not native:
        monkeypatch.setattr(_lib.host(), "norm_rope", lambda *a: NotImplemented)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)

    def strided(t):
        return torch.stack([t, t], -1)[..., 0]

    def gradients():
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, *weights)]
        return torch.autograd.grad(qk_norm_rope(*leaves[:2], positions, inv_freq, *leaves[2:]), leaves, (dq, dk))

    want = gradients()
    for back in (shifted, strided):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), back):
            assert all(torch.equal(a, b) for a, b in zip(gradients(), want)), back
