"""The operators between tokens and rows used together, as a training step and
as a decoding loop, and the ways a program calls them: on another stream, into
captured graphs (two of them replayed at once), at the same time on two
streams."""
import math

import pytest
import torch

import moderngpu_amd as m

pytestmark = pytest.mark.gpu


def test_training_step_with_a_tied_table(dev):
    """tokens -> rows -> logits against the same table -> distillation loss ->
    gradients.  The table's gradient is that of the logits' product, with the
    lookup's added onto it.  All values are 32-bit; the 64-bit reference is
    torch's autograd on the CPU.  Products of 48 and 37 terms, sums of 600 and
    64 terms: 2^-24 each, in all below 2^-13 of the largest gradient."""
    gen = torch.Generator().manual_seed(1)
    vocab, dim, tokens, top, tau = 600, 48, 64, 11, 2.0
    table = torch.randn(vocab, dim, generator=gen) * 0.3
    ids = torch.randint(-1, vocab, (tokens,), generator=gen).to(torch.int32)
    teacher_ids = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(tokens)]).to(torch.int32)
    teacher = torch.randn(tokens, top, generator=gen)
    weights = torch.rand(tokens, generator=gen) / tokens
    weights[::5] = 0

    w = table.double().requires_grad_()
    rows = torch.where((ids >= 0)[:, None], w[ids.long().clamp(min=0)] * 3.0, 0.0)
    log_q = torch.log_softmax(rows @ w.t() / tau, 1)
    p = torch.softmax(teacher.double() / tau, 1)
    want = (weights.double() * tau * tau * (p * (p.log() - log_q.gather(1, teacher_ids.long()))).sum(1)).sum()
    want.backward()

    t, i = table.to(dev), ids.to(dev)
    x = m.embedding_lookup(t, i, scale=3.0)
    loss, dz = m.distill_loss_and_grad(x @ t.t(), teacher_ids.to(dev), teacher.to(dev), temperature=tau, weights=weights.to(dev))
    grad = dz.t() @ x
    m.embedding_grad(dz @ t, i, scale=3.0, out=grad, accumulate=True)
    assert abs(loss.double().sum().item() - want.item()) <= 2.0 ** -13 * abs(want.item())
    assert (grad.double().cpu() - w.grad).abs().max() <= 2.0 ** -13 * w.grad.abs().max()


def test_decoding_loop(dev):
    """Draw a token a row, look its row up, add it to the state, and so on;
    greedy rows follow the largest logit.  Finished rows (-1) read zeros."""
    gen = torch.Generator().manual_seed(2)
    vocab, dim, rows = 500, 32, 6
    table = torch.randn(vocab, dim, generator=gen).to(dev)
    state = torch.randn(rows, dim, generator=gen).to(dev)
    temperature = torch.tensor([0.0, 1, 1, 0, 1, 1], device=dev)
    for step in range(8):
        logits = state @ table.t()
        logits[5] = -math.inf
        token, logprob = m.sample(logits, torch.rand(rows, generator=gen).to(dev), temperature=temperature, top_k=20, top_p=0.9)
        greedy = logits.argmax(1)
        assert token[0] == greedy[0] and token[3] == greedy[3] and token[5] == -1
        assert logprob[0] == 0 and logprob[5] == -math.inf and bool((logprob[:5] <= 0).all())
        kept = torch.topk(logits, 20, dim=1).indices
        assert bool((kept[:5] == token[:5, None]).any(1).all())
        row = m.embedding_lookup(table, token)
        assert torch.equal(row[:5], table[token[:5].long()]) and not row[5].any()
        state = torch.tanh(0.5 * state + 0.1 * row)


class Program:
    """Every entry point once, on buffers that stay."""

    def __init__(self, dev, seed, tokens=700, vocab=5003, dim=136):
        self.gen = torch.Generator().manual_seed(seed)
        self.table = torch.empty(vocab, dim, device=dev, dtype=torch.bfloat16)
        self.ids = torch.empty(tokens, dtype=torch.int32, device=dev)
        self.grad = torch.empty(tokens, dim, device=dev, dtype=torch.bfloat16)
        self.logits = torch.empty(40, vocab, device=dev)
        self.teacher_ids = torch.empty(40, 9, dtype=torch.int32, device=dev)
        self.teacher = torch.empty(40, 9, device=dev)
        self.weights = torch.ones(40, device=dev)
        self.uniform = torch.empty(40, device=dev)
        self.new_inputs()

    def new_inputs(self):
        g = self.gen
        for t in (self.table, self.grad, self.logits, self.teacher):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        self.ids.copy_(torch.randint(-3, self.table.shape[0], self.ids.shape, generator=g))
        self.ids[::4] = self.ids[0]
        self.teacher_ids.copy_(torch.randint(0, self.logits.shape[1], self.teacher_ids.shape, generator=g))
        self.uniform.copy_(torch.rand(40, generator=g))

    def run(self):
        rows = m.embedding_lookup(self.table, self.ids, scale=2.0)
        table_grad = m.embedding_grad(self.grad, self.ids, num_rows=self.table.shape[0])
        total = torch.zeros(self.table.shape, device=self.table.device)
        m.embedding_grad(self.grad, self.ids, out=total, accumulate=True)
        loss, norms = m.distill_loss(self.logits, self.teacher_ids, self.teacher, weights=self.weights)
        grad = m.distill_grad(self.logits, norms, self.teacher_ids, self.teacher, weights=self.weights)
        both = m.distill_loss_and_grad(self.logits, self.teacher_ids, self.teacher, weights=self.weights)
        all_kept = m.sample(self.logits, self.uniform)
        some = m.sample(self.logits, self.uniform, top_k=30, top_p=0.8, min_p=0.01)
        one = m.sample(self.logits[:1], self.uniform[:1], top_p=0.9)
        return [rows, table_grad, total, loss, norms, grad, *both, *all_kept, *some, *one]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


def test_calls_on_another_stream(dev):
    p = Program(dev, 3)
    want = p.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = p.run()
    side.synchronize()
    assert same(got, want)


def test_calls_on_two_streams_at_once(dev):
    programs = [Program(dev, 4), Program(dev, 5)]
    want = [p.run() for p in programs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(programs[i].run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same(g, want[i]) for g in got[i])


def test_captured_calls_replay_with_new_inputs(dev):
    """Two graphs of all entry points, replayed several times with new inputs
    and eager calls in between, then both at once on two streams."""
    programs = [Program(dev, 6), Program(dev, 7)]
    graphs, outs = [], []
    for p in programs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            p.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(p.run())
        graphs.append(graph)
    for _ in range(4):
        for p, graph, out in zip(programs, graphs, outs):
            p.new_inputs()
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, p.run())
    for p in programs:
        p.new_inputs()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
            graph.replay()
    torch.cuda.synchronize()
    for p, out in zip(programs, outs):
        assert same(out, p.run())
