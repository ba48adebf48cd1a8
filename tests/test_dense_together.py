"""The dense operators as a program uses them: a ranking model's steps (loss and gradient, the orthogonalised update of the
item table) and its answers in 8 bits, eager, captured into graphs, and on two streams at once.  No result depends on
timing, so all of these are compared bit by bit."""
import pytest

import rsgpu  # noqa: F401  (the library is built)

torch = pytest.importorskip("torch")

U32 = 2.0 ** -24


class Model:
    def __init__(self, ctx, n, v, k, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        self.ctx = ctx
        self.H = (torch.randn(n, k, generator=g) / k ** 0.5).to(dtype).cuda()
        self.W = torch.randn(v, k, generator=g).to(dtype).cuda()
        self.bias = torch.randn(v, generator=g).cuda()
        self.bias[v // 3] = -torch.inf
        self.weight = torch.rand(n, generator=g).cuda()
        self.target = torch.randint(-1, v, (n,), generator=g, dtype=torch.int32).cuda()

    def step(self):
        self.loss, _, dH, dW, db = self.ctx.softmax_ce(self.H, self.W, self.target, bias=self.bias, weight=self.weight, grad=True)
        self.H.sub_(dH, alpha=0.5)
        self.W.sub_(self.ctx.orthogonalize(dW), alpha=0.02)
        self.bias.sub_(db, alpha=0.1)
        q, s = self.ctx.quantize_rows(self.W)
        h, r = self.ctx.quantize_rows(self.H)
        self.scores = self.ctx.i8_matmul(h, r, q, s, col_bias=self.bias)

    def state(self):
        return [t.clone() for t in (self.H, self.W, self.bias, self.loss, self.scores)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


SIZES = [(40, 300, 20, torch.float32), (257, 1001, 100, torch.float32), (300, 5000, 64, torch.bfloat16), (64, 700, 256, torch.float16)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,k,dtype", SIZES)
def test_steps_and_answers(ctx, n, v, k, dtype):
    m = Model(ctx, n, v, k, dtype, seed=n)
    for _ in range(3):
        m.step()
    assert torch.isfinite(m.loss).all() and torch.isfinite(m.W).all() and torch.isfinite(m.H).all()
    assert (m.scores[:, v // 3] == -torch.inf).all()
    # the answers within half a step of each row's quantiser
    H, W = m.H.double(), m.W.double()
    r, s = H.abs().amax(1, keepdim=True) / 127, W.abs().amax(1) / 127
    bound = (r * W.abs().sum(1) + H.abs().sum(1, keepdim=True) * s) / 2 + k * r * s / 4
    exact = H @ W.T + m.bias.double()
    there = torch.isfinite(m.bias)
    err, lim = (m.scores.double() - exact)[:, there].abs(), (bound * (1 + 1e-6) + 8 * U32 * (H.abs() @ W.abs().T + m.bias.double().abs()))[:, there]
    assert (err <= lim).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,k,dtype", SIZES)
def test_two_graphs_in_turn(ctx, n, v, k, dtype):
    """Two captured models, replayed in turn with eager work between, against the same steps without graphs."""
    eager = [Model(ctx, n, v, k, dtype, seed) for seed in (1, 2)]
    models = [Model(ctx, n, v, k, dtype, seed) for seed in (1, 2)]
    graphs = []
    for m in models:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            m.step()
        graphs.append(g)
    for turn in range(4):
        for e, m, g in zip(eager, models, graphs):
            g.replay()
            e.step()
            if turn % 2:
                torch.cuda.synchronize()
        assert all(same(e.state(), m.state()) for e, m in zip(eager, models))


@pytest.mark.gpu
def test_two_streams_at_once(ctx):
    sizes = [(300, 5000, 64, torch.bfloat16), (257, 3001, 100, torch.float32)]
    want = []
    for i, size in enumerate(sizes):
        m = Model(ctx, *size, seed=i)
        for _ in range(5):
            m.step()
        want.append(m.state())
    models = [Model(ctx, *size, seed=i) for i, size in enumerate(sizes)]
    streams = [torch.cuda.Stream() for _ in sizes]
    torch.cuda.synchronize()
    for _ in range(5):
        for m, s in zip(models, streams):
            with torch.cuda.stream(s):
                m.step()
    torch.cuda.synchronize()
    assert all(same(w, m.state()) for w, m in zip(want, models))
