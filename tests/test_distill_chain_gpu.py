"""A head trained from a teacher's alternatives, as the operators are used together: the teacher's logits
give alternatives, the student's states go through a norm and a projection, the divergence goes back to
the projection, the norm's weights and the states."""
import pytest
import torch

from strim_amd import loss, norm, ops
from test_streams_gpu import beside, same

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def inputs(R, K, V, M, dtype, seed=0):
    g = gen(seed)
    teacher = (2.0 * torch.randn(R, V, device="cuda", generator=g)).to(dtype)
    h = torch.randn(R, K, device="cuda", generator=g).to(dtype)
    nw = (1.0 + 0.1 * torch.randn(K, device="cuda", generator=g)).to(dtype)
    w = (K ** -0.5 * torch.randn(V, K, device="cuda", generator=g)).to(dtype)
    return teacher, h, nw, w


def plain(h, nw, w, ids, logprobs, T, tail):
    """The mean divergence in 64 bits."""
    y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * nw
    lq = torch.log_softmax(y @ w.t() / T, -1)
    t = logprobs.double()
    p = t.exp()
    at = lq.gather(1, ids.long())
    if not tail:
        p = p / p.sum(-1, keepdim=True)
        return (p * (p.log() - at)).sum(-1).mean()
    r = 1.0 - p.sum(-1)
    rest = lq.exp().scatter(1, ids.long(), 0.0).sum(-1)
    return ((p * (t - at)).sum(-1) + r * (r.log() - rest.log())).mean()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("R,K,V,M", [(7, 64, 501, 8), (200, 96, 3_001, 32)])
def test_gradients_through_the_chain(R, K, V, M, tail):
    print(f"[chain] R={R} K={K} V={V} M={M} tail={tail}", flush=True)
    T = 1.5
    teacher, h, nw, w = inputs(R, K, V, M, torch.float32)
    scores = ops.token_scores(teacher, top=M, temperature=T)
    vals, ids = teacher.topk(M, -1)
    assert torch.equal(scores.top_ids.long(), ids)  # (float32 draws: no ties among the first M)

    def chain(h, nw, w):
        return loss.distill_loss(norm.rms_norm(h, nw) @ w.t(), scores.top_ids, scores.top_logprobs, T, tail)

    leaves = [t.clone().requires_grad_() for t in (h, nw, w)]
    value = chain(*leaves)
    value.backward()
    exact = [t.double().cpu().requires_grad_() for t in (h, nw, w)]
    ref = plain(*exact, scores.top_ids.cpu(), scores.top_logprobs.cpu(), T, tail)
    ref.backward()
    # A logit is a sum of K products of numbers below 5 and 0.6, accumulated in float32: its error is below
    # K 2^-24 sum |y w| < 96 2^-24 10 = 6e-5, which moves a probability, and so a gradient, by as much of itself;
    # the norm's and the products' own roundings add a few 2^-24 K more.
    tol = 2e-4
    assert abs(value.item() - ref.item()) <= tol * max(1.0, abs(ref.item()))
    for got, want in zip(leaves, exact):
        d = (got.grad.double().cpu() - want.grad).abs().max()
        assert d <= tol * want.grad.abs().max(), float(d)
    # and against differences of the 64-bit loss, along a direction for each leaf
    for i in range(3):
        u = torch.randn(exact[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        e = 1e-4
        with torch.no_grad():
            plus, minus = ([t + s * e * u if j == i else t for j, t in enumerate(exact)] for s in (1, -1))
            args = scores.top_ids.cpu(), scores.top_logprobs.cpu(), T, tail
            slope = (plain(*plus, *args) - plain(*minus, *args)) / (2 * e)
        got = (leaves[i].grad.double().cpu() * u).sum()
        # (an entry's error is at most tol of the largest; the differences' own is O(e^2))
        bound = tol * float(exact[i].grad.abs().max() * u.abs().sum()) + 1e-6
        assert abs(float(got - slope)) <= bound


def step(teacher, h, nw, w, weights, M, ws=(None, None, None)):
    """The chain by the operators: alternatives, states' norm, logits, loss and gradients."""
    t = ops.token_scores(teacher, top=M, workspace=ws[0])
    y, rstd, _ = ops.norm(h, nw)
    logits = y @ w.t()
    value, d_logits, status = ops.distill_step(logits, t.top_ids, t.top_logprobs, weights, tail=True,
                                               workspace=ws[1])
    d_h, d_nw, _ = ops.norm_grad(h, nw, None, d_logits @ w, rstd, workspace=ws[2])
    after = ops.token_scores(logits, t.top_ids[:, :1].contiguous(), workspace=ws[0])
    return [t.top_ids, t.top_logprobs, value, status, d_logits, d_h, d_nw, after.logprobs, after.entropy]


@pytest.mark.parametrize("R,K,V", [(5, 256, 40_003), (130, 512, 6_001)])
def test_captured_chains_share_a_workspace(R, K, V):
    """Two graphs of one workspace, replayed in turn over changed inputs with other work between."""
    print(f"[chain] graphs R={R} K={K} V={V}", flush=True)
    M = 16
    dtype = torch.bfloat16
    weights = torch.full((R,), 1.0 / R, device="cuda")
    sizes = (ops.token_scores_workspace(R, V, M), ops.distill_workspace(R, V, M, True),
             ops.norm_workspace(R, K, True))
    ws = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in sizes]
    held = [inputs(R, K, V, M, dtype, seed) for seed in (1, 2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in held:  # (the products' libraries set themselves up outside a capture)
            step(*x, weights, M, ws)
    torch.cuda.current_stream().wait_stream(side)
    for x in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*x, weights, M, ws))
        graphs.append(g)
    for turn in range(4):
        for i in (0, 1):
            for a, b in zip(held[i], inputs(R, K, V, M, dtype, 10 * turn + i)):
                a.copy_(b)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for i in (0, 1):
            same(got[i], step(*held[i], weights, M))


@pytest.mark.parametrize("R,V,M", [(6, 50_001, 20), (300, 9_000, 64)])
def test_calls_on_a_given_stream(R, V, M):
    print(f"[chain] streams R={R} V={V} M={M}", flush=True)
    K = 1_030
    teacher, h, nw, _ = inputs(R, K, V, M, torch.bfloat16, 3)
    logits = (2.0 * torch.randn(R, V, device="cuda", generator=gen(4))).to(torch.bfloat16)
    mask = torch.randint(-2 ** 31, 2 ** 31, (R, (V + 31) // 32), device="cuda", generator=gen(5)).int()
    tokens = torch.randint(0, V, (R,), device="cuda", generator=gen(6)).int()
    ones, dy = torch.ones(R, device="cuda"), torch.randn_like(h)
    t = ops.token_scores(teacher, tokens, M, 0.7, mask)
    _, lse, rest, _ = ops.distill(logits, t.top_ids, t.top_logprobs, tail=True)
    _, rstd, mean = ops.norm(h, nw, nw, center=True)
    n = ops.token_scores_workspace(R, V, M), ops.distill_workspace(R, V, M, True), ops.norm_workspace(R, K, True, True)

    def scores(s, x, k, m):
        return list(ops.token_scores(x, k, M, 0.7, m, stream=s))

    def scores_grad(s, x, k, l, e, g):
        return [ops.token_scores_grad(x, k, l, e, g, g, stream=s)]

    def distill(s, x, i, p):
        return list(ops.distill(x, i, p, tail=True, stream=s))

    def distill_grad(s, x, i, p, l, r, g):
        return [ops.distill_grad(x, i, p, l, r, g, tail=True, stream=s)]

    def distill_step(s, x, i, p, g):
        return list(ops.distill_step(x, i, p, g, tail=True, stream=s))

    def forward(s, x, w):
        return list(ops.norm(x, w, w, center=True, stream=s))

    def backward(s, x, w, g, r, m):
        return list(ops.norm_grad(x, w, w, g, r, m, stream=s))

    at = (logits, t.top_ids, t.top_logprobs)
    for call, args in ((scores, (teacher, tokens, mask)), (scores_grad, (teacher, tokens, t.lse, t.entropy, ones)),
                       (distill, at), (distill_grad, (*at, lse, rest, ones)), (distill_step, (*at, ones)),
                       (forward, (h, nw)), (backward, (h, nw, dy, rstd, mean))):
        print(f"[chain] {call.__name__}", flush=True)
        same(beside(call, list(args), [max(b, 16) for b in n] + [4 * R, 2 * R * V, 2 * R * K]), call(None, *args))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_second_device():
    """On the second device with the first one current: the same bits."""
    R, K, V, M = 6, 512, 3_000, 16
    x, weights = inputs(R, K, V, M, torch.bfloat16), torch.full((R,), 0.5, device="cuda")
    ref = step(*x, weights, M)
    got = step(*(t.to("cuda:1") for t in x), weights.to("cuda:1"), M)
    same([t.cpu() for t in got], [t.cpu() for t in ref])


def test_a_row_broadcast_over_several():
    """Expanded rows (stride 0) through the differentiable forms: the gradient is the rows' sum."""
    V, M, R = 700, 8, 5
    teacher, *_ = inputs(R, 16, V, M, torch.float32)
    t = ops.token_scores(teacher, top=M)
    row = torch.randn(V, device="cuda", generator=gen(1))
    grads = []
    for wide in (lambda r: r.expand(R, V), lambda r: r.repeat(R, 1)):
        leaf = row.clone().requires_grad_()
        x = wide(leaf)
        s = loss.token_scores(x, t.top_ids[:, 0].contiguous(), top=2)
        value = (loss.distill_loss(x, t.top_ids, t.top_logprobs) + s.logprobs.sum() + s.entropy.sum()
                 + (norm.layer_norm(x) * teacher).sum())
        grads.append(torch.autograd.grad(value, leaf)[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("R", [130, 20_011])
def test_captured_loss_with_its_backward(R):
    """The mean over many rows, forward and backward in a graph, replayed over changed inputs."""
    V, M = 90, 6
    teacher, *_ = inputs(R, 16, V, M, torch.float32)
    x = torch.randn(R, V, device="cuda", generator=gen(1)).requires_grad_()
    t = ops.token_scores(teacher, top=M)
    ids, lps = t.top_ids.clone(), t.top_logprobs.clone()

    def both():
        value = loss.distill_loss(x, ids, lps, tail=True)
        return [value.detach(), *torch.autograd.grad(value, x)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    for turn in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(R, V, device="cuda", generator=gen(turn)))
            lps[turn::7] = float("-inf")  # (rows without alternatives: the mean's count changes)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        same(got, both())
        live = (lps > float("-inf")).any(1)
        rows = loss.distill_loss(x.detach(), ids, lps, tail=True, reduction="none")
        # (N float32 sums in a tree of depth below 20: 20 2^-24 relative, the weights' rounding as well)
        want = rows.double()[live].mean()
        assert abs(got[0].double() - want) <= 2e-6 * rows.double()[live].abs().mean()
