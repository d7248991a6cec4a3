"""The operators between a language model's matrix products run together, as a training step uses them: embedding,
layer norm, a matrix product with the table, log probabilities and their gradient, back through layer norm into the
table, clipping by the global norm. Compared with the same step in 64 bits by automatic differentiation; then captured
into graphs, on several streams and from several host threads."""
import threading

import pytest
import torch

from tests.lm_cases import info, randn

pytestmark = pytest.mark.gpu
N, VOCAB, COLS, EPS = 160, 500, 64, 1e-5


class Step:
    """One step in the type `dt`, all buffers allocated once; run() makes the library's calls on a stream."""

    def __init__(self, ops, dt, seed, most=0.5):
        self.ops, self.dt, self.most = ops, dt, most
        kind = {0: torch.float32, 1: torch.float64}[dt]
        self.table = (0.3 * randn(seed, VOCAB, COLS)).to(kind)
        self.gain, self.bias = (1 + 0.1 * randn(seed + 1, COLS)).to(kind), (0.1 * randn(seed + 2, COLS)).to(kind)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.tokens = torch.randint(0, VOCAB, (N,), device="cuda", generator=gen)
        self.targets = torch.randint(0, VOCAB, (N,), device="cuda", generator=gen)
        self.tokens[5], self.targets[9] = -1, -1
        self.g = torch.full((N,), -1.0 / N, device="cuda", dtype=kind)
        self.gh = torch.full((N,), 0.02 / N, device="cuda", dtype=kind)

        def new(*shape):
            return torch.empty(*shape, device="cuda", dtype=kind)
        self.e, self.z, self.logits, self.dlogits, self.dz, self.de = new(N, COLS), new(N, COLS), new(N, VOCAB), new(N, VOCAB), new(N, COLS), new(N, COLS)
        self.mean, self.inv = new(N), new(N)
        self.lp, self.h, self.top, self.lse = new(N), new(N), new(N), new(N)
        self.dtable, self.dgain, self.dbias, self.norm = new(VOCAB, COLS), new(COLS), new(COLS), new(1)
        self.ids, self.lps = torch.empty(N, 5, dtype=torch.int64, device="cuda"), new(N, 5)

    def run(self):
        o, dt, x = self.ops, self.dt, [None, torch.cuda.current_stream().cuda_stream]
        o.execEmbedding(dt, x, self.table, info(self.table), self.tokens, 2.0, self.e, info(self.e))
        o.execLayerNorm(dt, x, self.e, info(self.e), self.gain, self.bias, EPS, self.z, info(self.z), self.mean, self.inv, [1], 1)
        torch.matmul(self.z, self.table.t(), out=self.logits)
        o.execTokenLogProbs(dt, x, self.logits, info(self.logits), self.targets, 1.0, self.lp, self.h, self.top, self.lse, 5, self.ids, self.lps)
        o.execTokenLogProbsGrad(dt, x, self.logits, info(self.logits), self.targets, 1.0, self.top, self.lse, self.h, self.g, self.gh,
                                self.dlogits, info(self.dlogits))
        torch.matmul(self.dlogits, self.table, out=self.dz)
        torch.matmul(self.dlogits.t(), self.z, out=self.dtable)
        o.execLayerNormGrad(dt, x, self.e, info(self.e), self.gain, self.mean, self.inv, self.dz, info(self.dz), self.de, info(self.de),
                            self.dgain, self.dbias, [1], 1)
        o.execEmbeddingGrad(dt, x, self.tokens, 2.0, self.de, info(self.de), self.dtable, info(self.dtable), True)
        grads = [self.dtable, self.dgain, self.dbias]
        o.execClipByGlobalNorm(dt, x, grads, None, [t.numel() for t in grads], 3, self.most, self.norm)

    def results(self):
        return [t.clone() for t in (self.lp, self.h, self.ids, self.dtable, self.dgain, self.dbias, self.norm)]

    def truth(self):
        leaves = [t.double().detach().requires_grad_() for t in (self.table, self.gain, self.bias)]
        table, gain, bias = leaves
        e = table[self.tokens.clamp(min=0)] * 2.0 * (self.tokens >= 0).double()[:, None]
        h = (e - e.mean(1, keepdim=True)) / torch.sqrt(e.var(1, correction=0, keepdim=True) + EPS)
        log_p = torch.log_softmax((h * gain + bias) @ table.t(), 1)
        live = (self.targets >= 0).double()
        lp = log_p.gather(1, self.targets.clamp(min=0)[:, None])[:, 0] * live
        entropy = -(log_p.exp() * log_p).sum(1) * live
        (self.g.double() * lp + self.gh.double() * entropy).sum().backward()
        norm = torch.sqrt(sum((t.grad ** 2).sum() for t in leaves))
        factor = min(1.0, self.most / float(norm))
        return [lp.detach(), entropy.detach(), None] + [t.grad * factor for t in leaves] + [norm[None]]


@pytest.mark.parametrize("dt", [0, 1])
def test_a_step_equals_automatic_differentiation(ops, dt):
    s = Step(ops, dt, 3)
    torch.backends.cuda.matmul.allow_tf32 = False
    s.run()
    assert float(s.norm) > s.most                            # the step is clipped
    for got, want in zip(s.results(), s.truth()):
        if want is not None:
            # a chain of seven products and sums of up to 500 terms: 500 roundings and then some, of the norm of each result
            assert float((got.double() - want).norm()) <= 2000 * torch.finfo(got.dtype).eps * float(want.norm())


def test_captured_steps_share_nothing(ops):
    # two graphs captured one after the other on one stream, replayed at the same time on two others, many times
    steps = [Step(ops, 0, 11), Step(ops, 0, 12)]
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append(s.results())
    graphs = []
    side = torch.cuda.Stream()
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.run()
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(s.results(), w))
    # new inputs in the same buffers are followed
    steps[0].tokens.copy_(steps[1].tokens)
    steps[0].targets.copy_(steps[1].targets)
    torch.cuda.synchronize()
    graphs[0].replay()
    torch.cuda.synchronize()
    got = steps[0].results()
    steps[0].run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(steps[0].results(), got))


def test_steps_on_several_streams_and_threads(ops):
    steps = [Step(ops, 0, 20 + k) for k in range(4)]
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append(s.results())
        for t in (s.dtable, s.lp, s.z):
            t.fill_(float("nan"))
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    errors = []

    def work(k):
        try:
            # two threads queue on one stream, the others have their own
            with torch.cuda.stream(shared if k < 2 else torch.cuda.Stream()):
                for _ in range(10):
                    steps[k].run()
            torch.cuda.synchronize()
        except Exception as e:                     # noqa: BLE001 -- reported by the test's own thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for s, w in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(s.results(), w))


def test_a_first_call_may_be_captured(ops):
    # nothing has run on this stream before: scratch memory is made inside the capture
    x = [randn(1, 50000).float(), randn(2, 333).float()]
    norm, want = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    ops.execGlobalNorm(0, [None, torch.cuda.current_stream().cuda_stream], x, [50000, 333], 2, want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        ops.execGlobalNorm(0, [None, torch.cuda.current_stream().cuda_stream], x, [50000, 333], 2, norm)
    for _ in range(3):
        norm.zero_()
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, want)


def test_tensors_of_another_device_or_type_are_refused(ops):
    from libnd4j_b200.native_ops import Nd4jError
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(Nd4jError, match="not in device memory"):
        ops.execLayerNorm(0, None, x, info(x), None, None, 1e-5, x.cpu(), info(x), None, None, [1], 1)
    with pytest.raises(Nd4jError, match="holds"):
        ops.execLayerNorm(2, None, x, info(x), None, None, 1e-5, x, info(x), None, None, [1], 1)
    with pytest.raises(Nd4jError, match="must be dense"):
        ops.execLayerNorm(0, None, x, info(x), torch.zeros(7, device="cuda"), None, 1e-5, x, info(x), None, None, [1], 1)
    with pytest.raises(Nd4jError, match="holds"):
        ops.execEmbedding(0, None, x, info(x), torch.zeros(4, dtype=torch.int32, device="cuda"), 1.0, torch.zeros(4, 8, device="cuda"), info(x))
    with pytest.raises(Nd4jError, match="beyond the tensor's memory"):
        wide = torch.zeros(5, 8, device="cuda")
        ops.execLayerNorm(0, None, x, info(wide), None, None, 1e-5, wide, info(wide), None, None, [1], 1)
    with pytest.raises(Nd4jError, match="must be dense"):
        ops.execTokenLogProbs(0, None, x, info(x), torch.zeros(8, dtype=torch.int64, device="cuda")[::2], 1.0, torch.zeros(4, device="cuda"),
                              None, None, None)
