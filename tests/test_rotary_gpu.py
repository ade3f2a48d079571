"""GPU: rotary positions against their formula in 64 bits, forward and backward."""
import pytest
import torch

from tests.serving_reference import close, turn, turn_bound

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(M, seed, dtype, B, T, H, G, D, rot, interleaved, scale):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(B, T * G, H, D, generator=gen, device=DEV).to(dtype)
    k = torch.randn(B, T, H, D, generator=gen, device=DEV).to(dtype)
    return q, k, M.Rotary(M.rotary_frequencies(rot, device=DEV)[0], interleaved, scale), gen


def _check(got, x, positions, rotary, what, inverse=False):
    rot = 2 * rotary.inv_freq.numel()
    want = turn(x.double(), positions, rotary.inv_freq, rotary.interleaved, rotary.scale, inverse)
    close(got, want, turn_bound(x.double(), want, rot, rotary.interleaved, rotary.scale, got.dtype), what)
    assert torch.equal(got[..., rot:], x[..., rot:]), what


SIZES = [  # B, T, H, G, D, rot
    (1, 1, 1, 1, 64, 64), (2, 5, 3, 2, 64, 16), (1, 33, 5, 4, 128, 128), (3, 7, 1, 1, 128, 96), (2, 64, 4, 8, 64, 48),
    (1, 300, 2, 3, 128, 64), (37, 1, 8, 4, 128, 128), (1, 4097, 8, 1, 64, 32), (5, 2, 13, 5, 128, 112),
]


@pytest.mark.parametrize("B,T,H,G,D,rot", SIZES)
@pytest.mark.parametrize("dtype,interleaved,scale", [(torch.bfloat16, False, 1.0), (torch.float16, True, 1.25), (torch.bfloat16, True, 1.0), (torch.float16, False, 0.75)])
def test_forward_and_gradients(built_library, B, T, H, G, D, rot, dtype, interleaved, scale):
    import moda_b200 as M
    q, k, rotary, gen = _case(M, B + T, dtype, B, T, H, G, D, rot, interleaved, scale)
    at = torch.randint(0, 100000, (B, T), generator=gen, device=DEV)
    q.requires_grad_(); k.requires_grad_()
    yq, yk = M.rotary_embedding(q, k, rotary, positions=at, moda_group_num=G)
    assert M.last_launch_count() == 1
    gq, gk = (torch.randn(x.shape, generator=gen, device=DEV).to(dtype) for x in (q, k))
    dq, dk = torch.autograd.grad([yq, yk], [q, k], [gq, gk])
    for got, x, inverse, what in ((yq, q, False, "q"), (yk, k, False, "k"), (dq, gq, True, "dq"), (dk, gk, True, "dk")):
        _check(got.detach(), x.detach(), at, rotary, what, inverse)


# more tokens than warps run at once: two or four a warp, in steps
@pytest.mark.parametrize("B,T,H,G,D,rot", [(1, 10001, 1, 4, 64, 64), (3, 3335, 3, 3, 64, 32), (2, 4802, 4, 4, 64, 48), (1, 9999, 3, 2, 128, 128), (2, 2501, 2, 2, 128, 64)])
@pytest.mark.parametrize("dtype,interleaved,scale", [(torch.bfloat16, False, 1.0), (torch.float16, True, 1.25)])
def test_many_tokens_of_few_heads(built_library, B, T, H, G, D, rot, dtype, interleaved, scale):
    test_forward_and_gradients(built_library, B, T, H, G, D, rot, dtype, interleaved, scale)


@pytest.mark.parametrize("make", [
    lambda B, T: (None, torch.arange(T)), lambda B, T: (0, torch.arange(T)), lambda B, T: (12345, 12345 + torch.arange(T)),
    lambda B, T: (-3, torch.arange(T) - 3), lambda B, T: (torch.arange(T, dtype=torch.int32) * 3, torch.arange(T) * 3),
    lambda B, T: (torch.arange(T).expand(B, T) + 7, torch.arange(T) + 7), lambda B, T: ((torch.arange(T) - 5)[None], torch.arange(T) - 5),
    lambda B, T: (torch.arange(2 * T).view(T, 2).t()[1], 2 * torch.arange(T) + 1),
    lambda B, T: (torch.full((T,), 2 ** 31 - 1, dtype=torch.int32), torch.full((T,), 2 ** 31 - 1)),
])
def test_positions(built_library, make):
    import moda_b200 as M
    B, T, G = 3, 9, 2
    q, k, rotary, _ = _case(M, 1, torch.float16, B, T, 2, G, 64, 64, False, 1.0)
    given, want = make(B, T)
    if isinstance(given, torch.Tensor):
        given = given.to(DEV)
    yq, yk = M.rotary_embedding(q, k, rotary, positions=given, moda_group_num=G)
    at = want.to(DEV).expand(B, T)
    _check(yq, q, at, rotary, "q"), _check(yk, k, at, rotary, "k")


def test_far_positions_are_as_exact_as_near_ones(built_library):
    """A million and a thousand million positions out; fp32 angles would be off by whole turns there.  The 64-bit reference itself
    rounds p f to 2^-53 of it: 1e-7 radians at 10^9, within what the bound leaves for the angle."""
    import moda_b200 as M
    q, k, rotary, _ = _case(M, 2, torch.float16, 1, 64, 2, 1, 128, 128, True, 1.0)
    for start in (10 ** 6, 10 ** 9):
        yq, yk = M.rotary_embedding(q, k, rotary, positions=start)
        at = (start + torch.arange(64, device=DEV))[None]
        _check(yq, q, at, rotary, "q"), _check(yk, k, at, rotary, "k")


def test_strided_inputs_and_views(built_library):
    import moda_b200 as M
    B, N, H, G, D = 2, 19, 3, 2, 64
    qp, kvp = torch.randn(B, N, G * H * D, device=DEV).bfloat16(), torch.randn(B, N, 2 * H * D, device=DEV).bfloat16()
    q, k, _ = M.fold_qkv(qp, kvp, H, G)
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    at = torch.arange(N, device=DEV).expand(B, N)
    yq, yk = M.rotary_embedding(q, k, rotary, moda_group_num=G)
    _check(yq, q, at, rotary, "q"), _check(yk, k, at, rotary, "k")
    wide = torch.randn(B, 2 * N, H + 2, D + 8, device=DEV).bfloat16()
    for x in (wide[:, ::2, 1:-1, :D], wide[:, :N, 1:-1, 4 : D + 4], wide[:1, :N, :1, :D].expand(B, N, H, D), wide[:, :N, :H, :D].flip(1)):
        _check(M.rotary_embedding(x, None, rotary), x, at, rotary, "view")


def test_gradient_against_differences(built_library):
    """The map is linear: <g, R(x + h) - R(x)> = <R'g, h>.  Inputs and steps are small whole numbers, which bf16 holds exactly,
    and every output is rounded by half a step: the two sides differ by at most the sum of |g| times those roundings, and
    of |h| times those of R'g."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(3)
    B, T, H, G, D = 1, 11, 2, 2, 64
    rotary = M.Rotary(M.rotary_frequencies(32, device=DEV)[0], True, 1.5)
    whole = lambda *s: torch.randint(-8, 9, s, generator=gen, device=DEV).bfloat16()  # noqa: E731
    q, h, g = (whole(B, T * G, H, D) for _ in range(3))
    q.requires_grad_()
    y = M.rotary_embedding(q, None, rotary, positions=100, moda_group_num=G)
    dq, = torch.autograd.grad(y, q, g)
    with torch.no_grad():
        y1 = M.rotary_embedding(q + h, None, rotary, positions=100, moda_group_num=G)
    left = (g.double() * (y1.double() - y.detach().double())).sum()
    right = (dq.double() * h.double()).sum()
    step = torch.finfo(torch.bfloat16).eps / 2
    bound = (g.double().abs() * (y1.double().abs() + y.detach().double().abs()) * step).sum() + (h.double().abs() * dq.double().abs() * step).sum()
    assert abs(left - right) <= bound * 1.01 + 1e-3
    # the bound is of use: a gradient turned the wrong way is outside it
    wrong = turn(g.double(), 100 + torch.arange(T, device=DEV)[None], rotary.inv_freq, True, 1.5)
    assert abs(left - (wrong * h.double()).sum()) > bound


@pytest.mark.parametrize("which", ["q", "k", "only q needs it", "only k needs it", "k None"])
def test_partial_gradients(built_library, which):
    import moda_b200 as M
    G, T = 2, 6
    q, k, rotary, _ = _case(M, 4, torch.bfloat16, 2, T, 3, G, 64, 64, False, 1.0)
    q.requires_grad_(which != "only k needs it"); k.requires_grad_(which != "only q needs it")
    at = torch.arange(T, device=DEV).expand(2, T)
    if which == "k None":
        y = M.rotary_embedding(q, None, rotary, moda_group_num=G)
        g = torch.randn_like(y)
        _check(torch.autograd.grad(y, q, g)[0], g, at, rotary, "dq", True)
        return
    yq, yk = M.rotary_embedding(q, k, rotary, moda_group_num=G)
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    if which == "q":
        dq, dk = torch.autograd.grad(yq, [q, k], gq, allow_unused=True)
        _check(dq, gq, at, rotary, "dq", True)
        assert dk is None or not dk.any()
    elif which == "k":
        dq, dk = torch.autograd.grad(yk, [q, k], gk, allow_unused=True)
        _check(dk, gk, at, rotary, "dk", True)
        assert dq is None or not dq.any()
    elif which == "only q needs it":
        _check(torch.autograd.grad([yq, yk], [q], [gq, gk])[0], gq, at, rotary, "dq", True)
    else:
        _check(torch.autograd.grad([yq, yk], [k], [gq, gk])[0], gk, at, rotary, "dk", True)


def test_gradients_of_shared_and_expanded_inputs(built_library):
    """One key head for all query heads: the caller expands it, and its gradient is the heads' sum.  A gradient that arrives
    expanded (of a sum) is taken as it is."""
    import moda_b200 as M
    T, H, D = 5, 4, 64
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    q = torch.randn(1, T, H, D, device=DEV).half().requires_grad_()
    one = torch.randn(1, T, 1, D, device=DEV).half().requires_grad_()
    yq, yk = M.rotary_embedding(q, one.expand(1, T, H, D), rotary)
    dq, dk = torch.autograd.grad(yq.sum() + yk.sum(), [q, one])
    at = torch.arange(T, device=DEV)[None]
    ones = torch.ones(1, T, H, D, device=DEV, dtype=torch.float16)
    _check(dq, ones, at, rotary, "dq", True)
    want = turn(ones.double(), at, rotary.inv_freq, False, 1.0, True)
    tol = turn_bound(ones.double(), want, D, False, 1.0, torch.float16).sum(2, keepdim=True) + 3 * torch.finfo(torch.float16).eps / 2 * want.abs().sum(2, keepdim=True)
    close(dk, want.sum(2, keepdim=True), tol, "dk")


def test_second_derivative_is_the_rotation_again(built_library):
    import moda_b200 as M
    q, k, rotary, _ = _case(M, 5, torch.bfloat16, 1, 7, 2, 1, 64, 64, False, 1.0)
    q.requires_grad_()
    y = M.rotary_embedding(q, None, rotary)
    g = torch.randn_like(y).requires_grad_()
    dq, = torch.autograd.grad(y, q, g, create_graph=True)
    v = torch.randn_like(dq)
    dg, = torch.autograd.grad(dq, g, v)
    _check(dg, v, torch.arange(7, device=DEV)[None], rotary, "dg")


@pytest.mark.parametrize("which", ["positions", "inv_freq"])
def test_changed_positions_or_frequencies_are_noticed(built_library, which):
    import moda_b200 as M
    q, k, rotary, _ = _case(M, 6, torch.bfloat16, 1, 7, 2, 1, 64, 64, False, 1.0)
    q.requires_grad_()
    at = torch.arange(7, device=DEV)
    y = M.rotary_embedding(q, None, rotary, positions=at)
    (at if which == "positions" else rotary.inv_freq).add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals_on_the_gpu(built_library):
    import torch.autograd.forward_ad as fwAD

    import moda_b200 as M
    q, k, rotary, _ = _case(M, 7, torch.bfloat16, 1, 7, 2, 1, 64, 64, False, 1.0)
    with pytest.raises(AssertionError, match="share dtype and device"):
        M.rotary_embedding(q, k.half(), rotary)
    with pytest.raises(AssertionError, match="one device"):
        M.rotary_embedding(q, k, M.Rotary(rotary.inv_freq.cpu()))
    with pytest.raises(AssertionError, match="one device"):
        M.rotary_embedding(q, k, rotary, positions=torch.arange(7))
    with pytest.raises(TypeError, match="bf16/fp16"):
        M.rotary_embedding(q.float(), k.float(), rotary)
    with pytest.raises(NotImplementedError, match="inv_freq"):
        M.rotary_embedding(q, k, M.Rotary(rotary.inv_freq.clone().requires_grad_()))
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        M.rotary_embedding(fwAD.make_dual(q, torch.ones_like(q)), k, rotary)
    with pytest.raises(M.ModaLibraryError) as e:
        M.rotary_embedding(q[:0], k[:0], rotary)
    assert e.value.status == 2
    with pytest.raises(M.ModaLibraryError) as e:
        M.rotary_embedding(q[..., :32].contiguous(), None, M.Rotary(rotary.inv_freq[:8].clone()))
    assert e.value.status == 3


def test_captured_and_on_another_stream(built_library):
    """A captured training step follows new inputs and new positions."""
    import moda_b200 as M
    G, T = 2, 40
    q, k, rotary, _ = _case(M, 8, torch.bfloat16, 2, T, 3, G, 64, 64, False, 1.0)
    at = torch.arange(T, device=DEV).repeat(2, 1)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    q.requires_grad_(); k.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        yq, yk = M.rotary_embedding(q, k, rotary, positions=at, moda_group_num=G)
        return [yq.detach(), yk.detach(), *torch.autograd.grad([yq, yk], [q, k], [gq, gk])]

    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        q.copy_(torch.randn_like(q)); k.copy_(torch.randn_like(k)); gq.copy_(torch.randn_like(gq))
    at += 1000
    graph.replay()
    torch.cuda.synchronize()
    for got, x, inverse in zip(out, (q, k, gq, gk), (False, False, True, True)):
        _check(got, x.detach(), at, rotary, "captured", inverse)


def test_prompt_attention_with_positions(built_library):
    """As a block uses it: projections, positions, attention; gradients reach the projections."""
    import moda_b200 as M
    from oracle import moda_oracle as mo
    B, N, H, G, D, L = 1, 70, 2, 2, 64, 3
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    qp = torch.randn(B, N, G * H * D, device=DEV).bfloat16().requires_grad_()
    kvp = torch.randn(B, N, 2 * H * D, device=DEV).bfloat16().requires_grad_()
    kd, vd = (torch.randn(B, N * L, H, D, device=DEV).bfloat16() for _ in range(2))
    q, k, v = M.fold_qkv(qp, kvp, H, G)
    yq, yk = M.rotary_embedding(q, k, rotary, moda_group_num=G)
    o = M.parallel_moda(yq, yk, v, cached_k=kd, cached_v=vd, moda_group_num=G)
    do = torch.randn_like(o)
    got = torch.autograd.grad(o, [qp, kvp], do)
    at = torch.arange(N, device=DEV)[None]
    ref = mo.moda_attention_ref_grads(yq.detach().float().cpu(), yk.detach().float().cpu(), v.detach().float().cpu(), kd.float().cpu(), vd.float().cpu(), do.float().cpu(), None, G, mo.MODE_CAUSAL, 1)
    dq, dk = (turn(x.double(), at.cpu(), rotary.inv_freq.cpu(), False, 1.0, True) for x in (ref[2], ref[3]))
    want = (dq.reshape(B, N, -1), torch.stack([dk, ref[4].double()], 2).reshape(B, N, -1))
    for a, b in zip(got, want):
        assert ((a.cpu().double() - b).norm() / b.norm()).item() <= 5e-2      # the attention's own tolerance for gradients


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,base,factor", [(128, 1e4, 1.0), (128, 5e5, 8.0), (64, 1e7, 8.0)])
def test_slow_pairs_near_the_start(built_library, interleaved, D, base, factor):
    """Pairs (0, 1) turn to (-sin a, cos a), down to a = 2.1e-8: the angle is a small part of a turn, and its sine is to have as many significant
    digits as any other result.  bf16 rounds by half a step.  Before that, relative to the sine: the frequency in turns is cut at 2^-64
    of a turn, 2^-35 of the smallest here (3.3e-9 turns); the series leaves out 1e-11; the sine is rounded to 32 bits (2^-24), and its product with 1 is exact."""
    import moda_b200 as M
    inv_freq, _ = M.rotary_frequencies(D, base, "linear", factor, device=DEV)
    at = torch.tensor([[1, 2, 5, 33, 1000, -1]], device=DEV)
    x = torch.zeros(1, 6, 1, D, device=DEV, dtype=torch.bfloat16)
    first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, D // 2), slice(D // 2, D))
    x[..., second] = 1
    y = M.rotary_embedding(x, None, M.Rotary(inv_freq, interleaved), positions=at)
    a = at.double()[..., None, None] * inv_freq
    for got, want in ((y[..., first], -a.sin()), (y[..., second], a.cos())):
        # the reference rounds p f to 2^-53 of it: next to a zero of the function that is 2^-53 of a over the result
        close(got, want, (torch.finfo(torch.bfloat16).eps / 2 * (1 + 2.0 ** -20) + 2.0 ** -23) * want.abs() + 2.0 ** -52 * a.abs(), "slow pairs")
