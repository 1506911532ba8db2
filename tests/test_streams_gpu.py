"""Calls on a given stream: their temporary memory, inputs that the caller lets go of, and results
are safe from the caller's own stream. The given stream is busy when each call is queued, and memory of
every size that the call took is allocated and overwritten on the caller's stream before it starts."""
import pytest
import torch

from strim_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def bf16(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=gen(seed)).to(torch.bfloat16)


def beside(call, inputs, sizes):
    """call(stream, *inputs) queued behind other work, its inputs dropped, memory of these sizes
    (bytes) overwritten meanwhile; its results, copied on the caller's stream."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(40_000_000)
    mine = [None if t is None else t.clone() for t in inputs]
    sizes = sizes + [t.numel() * t.element_size() for t in inputs if t is not None]
    stream.wait_stream(torch.cuda.current_stream())
    out = call(stream, *mine)
    del mine
    held = [torch.empty(n, dtype=torch.uint8, device="cuda").fill_(0xFF) for n in sizes for _ in range(2)]
    torch.cuda.current_stream().wait_stream(stream)
    got = [None if t is None else t.clone() for t in out]
    # the results let go of while the caller's stream may still read them
    del out
    with torch.cuda.stream(stream):
        again = [torch.empty_like(t).zero_() for t in got if t is not None]
    torch.cuda.synchronize()
    del held, again
    return got


def same(got, ref):
    assert len(got) == len(ref)
    for a, b in zip(got, ref):
        assert (a is None and b is None) or torch.equal(a, b)


def loss_inputs(R, K, V):
    h, w = bf16(R, K, seed=1), bf16(V, K, seed=2) * K ** -0.5
    t = torch.randint(0, V, (R,), device="cuda", generator=gen(3)).to(torch.int32)
    return h, w, t


@pytest.mark.parametrize("R,K,V", [(5, 64, 700), (300, 512, 20_001)])
def test_loss_and_gradients(R, K, V):
    print(f"[streams] loss N={R} K={K} V={V}", flush=True)
    h, w, t = loss_inputs(R, K, V)
    ref = ops.head_loss(h, w, t)
    same(beside(lambda s, *a: ops.head_loss(*a, stream=s), (h, w, t),
                [ops.head_loss_workspace(R, K, V), 4 * R]), ref)
    gl = torch.randn(R, device="cuda", generator=gen(4))
    grads = ops.head_loss_grad(h, w, t, ref[1], gl)
    same(beside(lambda s, *a: ops.head_loss_grad(*a, stream=s), (h, w, t, ref[1], gl),
                [ops.head_loss_workspace(R, K, V, True, True), 2 * R * K, 2 * V * K]), grads)
    # a workspace of the caller's, let go of as well
    need = ops.head_loss_workspace(R, K, V, True, True)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    same(beside(lambda s, *a: ops.head_loss_grad(*a[:5], workspace=a[5], stream=s),
                (h, w, t, ref[1], gl, ws), [2 * R * K, 2 * V * K]), grads)


@pytest.mark.parametrize("B,K,V", [(3, 256, 1000), (20, 1024, 9000)])
def test_packed_weights(B, K, V):
    print(f"[streams] packed B={B} K={K} V={V}", flush=True)
    w, x = bf16(V, K, seed=5), bf16(B, K, seed=6)
    nw = bf16(K, seed=7)
    q = ops.q4_pack(w, 64)

    def parts(q):
        return q.words, q.scales, q.biases

    same(beside(lambda s, a: parts(ops.q4_pack(a, 64, stream=s)), (w,), [V * K // 2, V * K // 32]), parts(q))
    same(beside(lambda s, *a: (ops.q4_unpack(ops.Q4Weight(*a, 64), stream=s),), parts(q), [2 * V * K]),
         (ops.q4_unpack(q),))
    same(beside(lambda s, x, nw, *a: (ops.head_logits_q4(x, ops.Q4Weight(*a, 64), nw, stream=s),),
                (x, nw, *parts(q)), [2 * B * V, 2 * B * K, max(1, ops.head_logits_q4_workspace(B, K))]),
         (ops.head_logits_q4(x, q, nw),))


def test_dense_logits(ctx):
    B, K, V = 8, 512, 4096
    w, x, nw = bf16(V, K, seed=8), bf16(B, K, seed=9), bf16(K, seed=10)
    same(beside(lambda s, *a: (ops.head_logits(*a, stream=s),), (x, w, nw), [2 * B * V, 2 * B * K]),
         (ops.head_logits(x, w, nw),))
    same(beside(lambda s, *a: ops.head_greedy(ctx, *a, stream=s), (x, w, nw), [2 * B * K, 4 * B]),
         ops.head_greedy(ctx, x, w, nw))


def test_results_of_the_current_stream_given_by_name():
    """The current stream given explicitly: as without it."""
    h, w, t = loss_inputs(9, 64, 300)
    same(ops.head_loss(h, w, t, stream=torch.cuda.current_stream()), ops.head_loss(h, w, t))
