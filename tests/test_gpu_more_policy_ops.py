"""Layer norm, the gated delta rule and the drawing of actions as a policy runs
them: one after the other in a captured training step, from threads that run at
the same time, and in two graphs that are replayed in turn."""

from __future__ import annotations

import threading

import pytest
import torch

from .conftest import require_gpu

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


class _Net:
    """A norm, a memory and a head over features [steps, envs, heads * values], with leaves of its own."""

    def __init__(self, seed, steps, envs, heads, keys, values, dtype, share=1, actions=11):
        gen = _gen(seed)
        self.x = _randn(gen, steps, envs, heads * values, dtype=dtype)
        self.q = _randn(gen, steps, envs, heads // share, keys, dtype=dtype)
        self.k = _randn(gen, steps, envs, heads // share, keys, dtype=dtype)
        self.g = -0.05 - 0.2 * torch.rand(steps, envs, heads, device="cuda", generator=gen)
        self.beta = torch.sigmoid(_randn(gen, steps, envs, heads))
        self.resets = torch.rand(steps, envs, device="cuda", generator=gen) < 0.1
        self.weight, self.bias = 1 + _randn(gen, heads * values, scale=0.1), _randn(gen, heads * values, scale=0.1)
        self.head = _randn(gen, heads * values, actions, dtype=dtype, scale=0.2)
        self.uniform = torch.rand(envs, device="cuda", generator=gen)
        self.dy = _randn(gen, steps, envs, heads * values, dtype=dtype)
        self.shape = (steps, envs, heads, values)

    def leaves(self):
        return [t.detach().requires_grad_() for t in (self.x, self.q, self.k, self.g, self.beta, self.weight, self.bias)]

    def run(self, leaves):
        """Outputs and gradients, the drawn actions among them."""
        from gbxcule_amd.rl import delta_rule, layer_norm, sample_actions

        x, q, k, g, beta, weight, bias = leaves
        y = layer_norm(x, weight, bias)
        m, last = delta_rule(q, k, y.view(self.shape), g, beta, resets=self.resets)
        z, s = layer_norm(m.reshape(x.shape), weight, bias, x)
        with torch.no_grad():
            action, logp = sample_actions(z[-1] @ self.head, self.uniform, top_k=7, top_p=0.9)
        return [z.detach(), s.detach(), last, action, logp, *torch.autograd.grad(z, leaves, self.dy)]


# sizes whose gradient holds little and much in LDS, heads that share rows, and a forward pass in pieces
NETS = [
    (1, 20, 5, 2, 32, 24, BF16, 1),
    (2, 33, 3, 4, 24, 16, F32, 2),
    (3, 18, 2, 2, 128, 128, BF16, 1),
    (4, 400, 1, 1, 32, 32, F32, 1),
]


@pytest.mark.parametrize("net", NETS, ids=lambda n: f"{n[1]}x{n[2]}x{n[3]}_{n[4]}x{n[5]}")
def test_a_captured_training_step(net):
    n = _Net(*net)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # libraries set themselves up outside of the graph; nothing of this lives on
        n.run(n.leaves())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    fixed = n.leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = n.run(fixed)
    for turn in range(3):
        with torch.no_grad():
            for t in (n.x, n.q, n.k):
                t.copy_(_randn(_gen(100 + turn), *t.shape, dtype=t.dtype))
            n.uniform.copy_(torch.rand(n.uniform.shape, device="cuda", generator=_gen(200 + turn)))
        graph.replay()
        torch.cuda.synchronize()
        want = n.run(n.leaves())
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_two_graphs_in_turn():
    """Graphs of one memory pool, whose work buffers may lie at the same place, replayed one after the other."""
    nets = [_Net(*NETS[3]), _Net(*NETS[1])]
    from gbxcule_amd.rl import delta_rule, layer_norm, sample_actions

    def forward(n):
        y = layer_norm(n.x, n.weight, n.bias)
        m, last = delta_rule(n.q, n.k, y.view(n.shape), n.g, n.beta, resets=n.resets)
        return [m, last, *sample_actions(m[-1].flatten(1) @ n.head, n.uniform, top_p=0.8)]

    for n in nets:
        forward(n)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for n in nets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(forward(n))
        graphs.append(graph)
    for turn in range(3):
        for n, graph, out in zip(nets, graphs, outs):
            n.q.copy_(_randn(_gen(300 + turn), *n.q.shape, dtype=n.q.dtype))
            graph.replay()
            kept = [t.clone() for t in out]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, forward(n))), turn


def test_threads():
    """Four threads, each on a stream of its own, as actors beside a learner."""
    nets = [_Net(*n) for n in NETS]
    want = [n.run(n.leaves()) for n in nets]
    torch.cuda.synchronize()
    wrong, done = [], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = nets[i].run(nets[i].leaves())
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
            done.append(i)
        except Exception as e:  # a thread's own exception would be lost
            wrong.append((i, e))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(nets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(done) == len(nets), wrong


def test_offsets_past_32_bits():
    """More than 2^31 elements: what is at the end equals the same rows by themselves, bit for bit."""
    from gbxcule_amd.rl import delta_rule, delta_rule_step, layer_norm, sample_actions

    gen = _gen(9)
    some = lambda *shape, dtype=BF16: torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)  # noqa: E731
    # layer norm and drawing, a row each
    x = some(1_100_000, 2000)
    w, b = 1 + 0.1 * some(2000, dtype=F32), some(2000, dtype=F32)
    assert torch.equal(layer_norm(x, w, b)[-700:], layer_norm(x[-700:].clone(), w, b))
    u = torch.rand(1_100_000, device="cuda", generator=gen)
    for got, want in zip(sample_actions(x, u, top_k=30), sample_actions(x[-700:].clone(), u[-700:], top_k=30)):
        assert torch.equal(got[-700:], want)
    leaf, part = x.requires_grad_(), x[-700:].detach().clone().requires_grad_()
    dy = some(700, 2000)
    wide = torch.zeros_like(x)
    wide[-700:] = dy
    (found,) = torch.autograd.grad(layer_norm(leaf, w, b), [leaf], wide)
    assert torch.equal(found[-700:], torch.autograd.grad(layer_norm(part, w, b), [part], dy)[0])
    del x, leaf, found, wide
    # the delta rule: 33 x 8,192 x 64 heads of 8 x 128, of whose envs the last 64 alone make as many wavefronts a compute unit
    q, k, v = some(33, 8192, 64, 8), some(33, 8192, 64, 8), some(33, 8192, 64, 128)
    g, beta = -0.1 * torch.rand(33, 8192, 64, device="cuda", generator=gen), torch.rand(33, 8192, 64, device="cuda", generator=gen)
    rows = [q, k, v, g, beta]
    last = lambda t: t[:, -64:].clone()  # noqa: E731
    whole, part = [t.requires_grad_() for t in rows], [last(t.detach()).requires_grad_() for t in rows]
    y, s = delta_rule(*whole)
    y2, s2 = delta_rule(*part)
    assert torch.equal(y[:, -64:], y2) and torch.equal(s[-64:], s2)
    dy = some(33, 8192, 64, 128)
    for got, want in zip(torch.autograd.grad(y, whole, dy), torch.autograd.grad(y2, part, last(dy))):
        assert torch.equal(got[:, -64:], want)
    del whole, part, y, dy, rows, got, want
    # a step, with more than 2^31 numbers of state
    state = some(33_000, 16, 64, 64, dtype=F32)
    kept = state[-64:].clone()
    rows = [some(33_000, 16, 64) for _ in range(3)] + [g.detach().flatten()[: 33_000 * 16].view(33_000, 16), beta.detach().flatten()[: 33_000 * 16].view(33_000, 16)]
    y = delta_rule_step(*rows, state=state)
    assert torch.equal(y[-64:], delta_rule_step(*(t[-64:].clone() for t in rows), state=kept)) and torch.equal(state[-64:], kept)
