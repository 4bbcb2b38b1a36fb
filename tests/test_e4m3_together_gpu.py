"""The quantised cache's operators one after the other, as a step uses them: on a stream, on two streams at once, in a graph that is
replayed over other numbers."""

import pytest
import torch

from . import e4m3_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from shrike_amd.kernels import ops

    return ops


class Cached:
    """A step of single tokens and portions after it, over a cache that is filled token by token of its starts, all on the device."""

    def __init__(self, ops, form, starts, news, seed):
        self.ops, self.form = ops, form
        heads, kv, dim, ps = form
        self.plan = plain.Step(starts, news, ps, seed=seed)
        self.singles = sum(1 for n in news if n == 1)
        step = self.plan
        self.width = (heads + 2 * kv) * dim
        k, v, s, self.keys, self.values = plain.random_pools(step.pages, kv, dim, ps, step.gen)
        self.start = [k.cuda(), v.cuda(), s.cuda()]
        self.pools = [torch.empty_like(x) for x in self.start]
        self.rows = torch.randn(step.n, self.width, generator=step.gen).bfloat16()
        self.qkv = self.rows.cuda()
        self.q = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
        self.inv_freq = (10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float()
        self.args = [x.cuda() for x in (self.inv_freq, step.positions, step.token_seq, step.tables, step.cu_q, step.ctx_lens)]
        self.out = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
        self.back = [torch.empty(step.n, kv * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.partial = torch.empty(step.n * heads * 3 * (dim + 2), device="cuda")

    def run(self):
        heads, kv, dim, ps = self.form
        freq, positions, seqs, tables, cu_q, ctx_lens = self.args
        ops, scale = self.ops, dim ** -0.5
        for to, start in zip(self.pools, self.start):
            to.view(torch.uint8).copy_(start.view(torch.uint8))
        self.out.zero_()
        ops.rope_kv_store_e4m3(self.qkv, heads, kv, dim, dim, freq, positions, seqs, tables, *self.pools, ps, q_out=self.q)
        ops.attention_decode_e4m3(self.q, self.out, self.singles, heads, kv, dim, positions, tables, *self.pools, ps, None, scale,
                                  self.partial, 3)
        ops.attention_prefill_e4m3(self.q, self.out, self.singles, len(self.plan.news) - self.singles, heads, kv, dim, cu_q, ctx_lens, tables,
                                   *self.pools, ps, None, scale, self.partial, 2)
        ops.kv_read_e4m3(*self.back, kv, dim, positions, seqs, tables, *self.pools, ps)

    def results(self):
        return [x.view(torch.uint8).clone() for x in (self.out, self.q, *self.back, *self.pools)]

    def check(self):
        """Results against 64 bits, from the codes that the step has left (how they are chosen is tested by itself)."""
        heads, kv, dim, ps = self.form
        step = self.plan
        keys, values = self.keys.clone(), self.values.clone()
        slots = step.positions.long() % ps
        pages = step.tables[step.token_seq.long(), step.positions.long() // ps].long()
        for paged, rows in zip((keys, values), self.back):
            paged[pages, :, slots] = rows.cpu().double().view(step.n, kv, dim)
        raw = self.qkv.cpu().double().view(step.n, heads + 2 * kv, dim)
        turned = plain.rotate(raw[:, :heads + kv], step.positions, self.inv_freq, dim)
        for at, rows in ((heads, turned[:, heads:]), (0, raw[:, heads + kv:])):
            have = self.back[0 if at else 1].cpu().double().view(step.n, kv, dim)
            unit = torch.ldexp(torch.ones_like(rows[..., :1]), plain.exponents(rows)[..., None])
            # half a step of the code (of twice the size where rounding has moved the power of two), and the turn in float32
            assert ((have - rows).abs() <= 2 * plain.half_step(rows / unit) * unit * (1 + 2.0 ** -10)).all()
        want, size, reach = plain.attention(step, self.q.cpu(), keys, values, heads, dim ** -0.5)
        limit = plain.allowed(want, size, reach, dim, max(step.ctx_lens.tolist()), True)
        assert ((self.out.cpu().double().view_as(want) - want).abs() <= limit).all()


FORMS = [(14, 2, 64, 16), (28, 4, 128, 16), (8, 2, 128, 64), (8, 1, 256, 32)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("starts, news", [([0, 33], [1, 1]), ([200, 5, 0, 70], [1, 1, 90, 17]), ([64], [100])])
def test_a_step(ops, form, starts, news):
    step = Cached(ops, form, starts, news, 1)
    step.run()
    step.check()


@pytest.mark.parametrize("form", FORMS[:2])
def test_two_streams_at_once(ops, form):
    steps = [Cached(ops, form, [700, 30, 0], [1, 1, 200], 2), Cached(ops, form, [900, 0, 100], [1, 1, 150], 3)]
    alone = []
    for step in steps:
        step.run()
        alone.append(step.results())
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(5):
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step.run()
    torch.cuda.synchronize()
    for step, want in zip(steps, alone):
        assert all(torch.equal(a, b) for a, b in zip(step.results(), want))
        step.check()


@pytest.mark.parametrize("form", FORMS)
def test_a_graph_replayed_over_other_numbers(ops, form):
    """Positions, lengths, tables and rows change between replays, as eager work on the same workspace does."""
    step = Cached(ops, form, [300, 90, 150], [1, 1, 80], 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    ps = form[3]
    for round_, starts in enumerate(([300, 90, 150], [17, 200, 0], [299, 0, 151], [0, 1, 2], [301, 90, 150])):
        step.plan.starts = starts
        step.plan.ctx_lens = torch.tensor([a + n for a, n in zip(starts, step.plan.news)], dtype=torch.int32)
        if max(-(-int(n) // ps) for n in step.plan.ctx_lens) > step.plan.tables.shape[1] or any(
                int(step.plan.tables[i, -(-int(n) // ps) - 1]) < 0 for i, n in enumerate(step.plan.ctx_lens)):
            continue  # (more pages than these tables have)
        step.plan.positions = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, step.plan.news)]).to(torch.int32)
        step.args[1].copy_(step.plan.positions)
        step.args[5].copy_(step.plan.ctx_lens)
        step.rows = torch.randn(step.rows.shape, generator=step.plan.gen).bfloat16()
        step.qkv.copy_(step.rows)
        step.run()
        want = step.results()
        step.partial.fill_(float("nan"))
        step.out.fill_(7.0)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step.results(), want)), f"replay {round_}"
        step.check()
