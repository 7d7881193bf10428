"""The paged cache, shared-prefix attention and sampling as a program runs
them together: a prompt into the shared pages, ragged questions behind it,
then one token at a time fed back to the cache, eagerly and as one captured
graph that counts its own lengths up.

The model is one attention layer whose projections are tables: a row of qkv
and a row of output logits per token id.

Tolerance of a step's attention against 64 bits, from the tokens' own rows: q,
k and v are rounded once each to the cache's type (half a step h), so a score
is off by at most d = (2 h + h^2 + 2^-16) sum |q k| (2^-16: the f32 rotation and
sums) and a probability by a factor e^(2 d); v, the probabilities and the output
add a half step each, the f32 sums over keys 2^-17 of sum p |v|."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import ELEM, TYPES, half_step, plain_rope, rope_table
from test_sample_gpu import plain as plain_sample

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

VOCAB, STEPS = 1500, 6


class Decoder:
    """A pool of pages, the model's tables and the buffers of each step."""

    def __init__(self, seed, nseq, prefix, heads, kv_heads, hd, dtype, window, temperature, top_k, top_p, page=16):
        rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.hd, self.dtype, self.window = heads, kv_heads, hd, dtype, window
        self.width, self.prefix, self.nseq, self.page = (heads + 2 * kv_heads) * hd, prefix, nseq, page
        self.questions = [rng.integers(0, VOCAB, int(n)) for n in rng.integers(1, 41, nseq)]
        self.prompt = rng.integers(0, VOCAB, prefix)
        f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()
        self.qkv_of, self.head = f(VOCAB, self.width), f(heads * hd, VOCAB) * 0.4
        most = -(-(40 + STEPS) // page)
        pre = -(-prefix // page)
        ids = rng.permutation(pre + nseq * most).astype(np.int32)
        self.prefix_table = torch.from_numpy(ids[:pre].copy()).cuda()
        self.table = torch.from_numpy(ids[pre:].reshape(nseq, most).copy()).cuda()
        self.max_pages = most
        self.k, self.v = (torch.full((len(ids), kv_heads, page, hd), float("nan"), device="cuda").to(TYPES[dtype])
                          for _ in range(2))
        self.kv = g.PagedKv(self.k.data_ptr(), self.v.data_ptr(), len(ids), kv_heads, page, hd, ELEM[dtype])
        self.rope = rope_table(prefix + 40 + STEPS, hd).cuda()
        self.tokens = torch.zeros(nseq, dtype=torch.int32, device="cuda")
        self.logprob = torch.zeros(nseq, device="cuda")
        self.lens = torch.zeros(nseq, dtype=torch.int32, device="cuda")
        self.u = torch.zeros(nseq, device="cuda")
        par = lambda v, t: torch.from_numpy(np.resize(np.asarray(v, t), nseq)).cuda()
        self.temperature, self.top_p = par(temperature, np.float32), par(top_p, np.float32)
        self.top_k = par(top_k, np.int32)
        self.logits = torch.zeros(nseq, VOCAB, device="cuda")
        self.sample_ws = torch.full((g.sample_workspace(nseq, VOCAB) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        self.step_batch = g.PagedBatch(nseq, nseq, self.lens.data_ptr(), self.table.data_ptr(), most, None,
                                       self.prefix_table.data_ptr(), prefix)
        self.step_buffers = self.buffers(self.step_batch, nseq)

    def buffers(self, batch, rows):
        e = lambda *s: torch.empty(*s, dtype=TYPES[self.dtype], device="cuda")
        ws = torch.full((self.kv.attention_workspace(batch, self.heads) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        return e(rows, self.heads * self.hd), e(rows, self.heads * self.hd), ws

    def layer(self, batch, qkv, bufs):
        """Rows of qkv into the cache and through attention; the outputs."""
        q, out, ws = bufs
        stream = torch.cuda.current_stream().cuda_stream
        x, size = qkv.data_ptr(), qkv.element_size()
        self.kv.append(batch, g.KvSource(g.ELEM_F32, self.heads, x, x + self.heads * self.hd * size,
                                         x + (self.heads + self.kv_heads) * self.hd * size, self.width,
                                         rope=self.rope.data_ptr(), rope_rows=self.rope.shape[0], rope_dims=self.hd,
                                         q_scale=self.hd ** -0.5), q.data_ptr(), self.heads * self.hd, stream)
        self.kv.attention(batch, self.heads, q.data_ptr(), self.heads * self.hd, out.data_ptr(), self.heads * self.hd,
                          1.0, window=self.window, workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream)
        return out

    def draw(self, last):
        torch.mm(last.float(), self.head, out=self.logits)
        g.sample(self.logits.data_ptr(), g.ELEM_F32, self.nseq, VOCAB, VOCAB, self.u.data_ptr(), self.tokens.data_ptr(),
                 self.logprob.data_ptr(), temperature=self.temperature.data_ptr(), top_k=self.top_k.data_ptr(),
                 top_p=self.top_p.data_ptr(), workspace=self.sample_ws.data_ptr(),
                 workspace_bytes=self.sample_ws.numel(), stream=torch.cuda.current_stream().cuda_stream)

    def read_prompt(self):
        """The prompt as a batch of one sequence whose own pages are the shared ones."""
        if not self.prefix:
            return None
        n = torch.tensor([self.prefix], dtype=torch.int32, device="cuda")
        start = torch.tensor([0, self.prefix], dtype=torch.int32, device="cuda")
        b = g.PagedBatch(1, self.prefix, n.data_ptr(), self.prefix_table.data_ptr(), self.prefix_table.numel(),
                         start.data_ptr())
        qkv = self.qkv_of[torch.from_numpy(self.prompt).cuda()]
        out = self.layer(b, qkv, self.buffers(b, self.prefix))
        torch.cuda.synchronize()
        return out.double().cpu()

    def read_questions(self):
        counts = np.array([len(x) for x in self.questions])
        start = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
        self.lens.copy_(torch.from_numpy(counts.astype(np.int32)))
        t = int(counts.sum())
        b = g.PagedBatch(self.nseq, t, self.lens.data_ptr(), self.table.data_ptr(), self.max_pages, start.data_ptr(),
                         self.prefix_table.data_ptr(), self.prefix)
        qkv = self.qkv_of[torch.from_numpy(np.concatenate(self.questions)).cuda()]
        out = self.layer(b, qkv, self.buffers(b, t))
        self.draw(out[start[1:].long() - 1])
        torch.cuda.synchronize()
        return out.double().cpu(), start.cpu().numpy()

    def step(self):
        """One token of every sequence: the drawn ones go into the cache, the next are drawn."""
        self.lens.add_(1)
        qkv = self.qkv_of.index_select(0, self.tokens)
        out = self.layer(self.step_batch, qkv, self.step_buffers)
        self.draw(out)

    # The plain form.

    def attend(self, ids, rows):
        """Rows `rows` of a sequence of token ids through the layer in 64 bits: outputs and their bounds."""
        H, K, D = self.heads, self.kv_heads, self.hd
        x = self.qkv_of.double().cpu()[torch.from_numpy(np.asarray(ids))].view(len(ids), H + 2 * K, D)
        cs = self.rope.double().cpu()
        rot = lambda y: torch.stack([plain_rope(y[i], cs[i], g.ROPE_HALF) for i in range(len(y))])
        qr = torch.stack([plain_rope(x[i, :H], cs[i], g.ROPE_HALF) for i in rows]) * D ** -0.5
        k, v = rot(x[:, H:H + K]), x[:, H + K:]
        h = half_step(TYPES[self.dtype])
        at, key = torch.from_numpy(np.asarray(rows)), torch.arange(len(ids))
        see = key[None] <= at[:, None]
        if self.window:
            see &= key[None] > at[:, None] - self.window
        out, tol = torch.empty(len(rows), H, D, dtype=torch.float64), torch.empty(len(rows), H, D, dtype=torch.float64)
        for i in range(H):
            kh, vh = k[:, i // (H // K)], v[:, i // (H // K)]
            p = (qr[:, i] @ kh.T).masked_fill(~see, -np.inf).softmax(-1)
            d = (2 * h + h * h + 2.0 ** -16) * (qr[:, i].abs() @ kh.abs().T).masked_fill(~see, 0).amax(-1, keepdim=True)
            out[:, i] = p @ vh
            tol[:, i] = (p @ vh.abs()) * (torch.expm1(2 * d) + 3 * h + 2.0 ** -17)
        return out.reshape(len(rows), -1), tol.reshape(len(rows), -1)

    def check_rows(self, what, got, ids, rows):
        exp, tol = self.attend(ids, rows)
        bad = (got - exp).abs() > tol
        assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - exp).abs().max())}"

    def check_draw(self, what):
        z = self.logits.double().cpu().numpy()
        for s in range(self.nseq):
            t, l = plain_sample(z[s], float(self.u[s]), float(self.temperature[s]), int(self.top_k[s]), float(self.top_p[s]))
            assert int(self.tokens[s]) == t, f"{what}: sequence {s}"
            assert abs(float(self.logprob[s]) - l) <= 2.0 ** -23 * max(1.0, abs(l)) + VOCAB * 2.0 ** -42


MODELS = [dict(nseq=5, prefix=77, heads=4, kv_heads=1, hd=256, dtype="bf16", window=0),
          dict(nseq=3, prefix=0, heads=15, kv_heads=5, hd=64, dtype="f16", window=0),
          dict(nseq=9, prefix=200, heads=8, kv_heads=2, hd=128, dtype="f16", window=60),
          dict(nseq=1, prefix=33, heads=2, kv_heads=2, hd=512, dtype="bf16", window=0)]
DRAWS = dict(temperature=[0.0, 0.8, 1.2, 1.5], top_k=[0, 40, 0, 300], top_p=[1.0, 1.0, 0.9, 0.95])


@pytest.mark.parametrize("m", range(len(MODELS)))
def test_prompt_questions_and_tokens_one_at_a_time(m):
    d = Decoder(100 + m, **MODELS[m], **DRAWS)
    rng = np.random.default_rng(m)
    rows = d.read_prompt()
    if rows is not None:
        d.check_rows("prompt", rows, d.prompt, np.arange(d.prefix))
    d.u.copy_(torch.from_numpy(rng.random(d.nseq).astype(np.float32)))
    out, start = d.read_questions()
    ids = [np.concatenate([d.prompt, x]) for x in d.questions]
    for s in range(d.nseq):
        d.check_rows(f"question {s}", out[start[s]:start[s + 1]], ids[s], np.arange(d.prefix, len(ids[s])))
    d.check_draw("questions")
    for n in range(STEPS):
        ids = [np.append(x, t) for x, t in zip(ids, d.tokens.cpu().numpy())]
        d.u.copy_(torch.from_numpy(rng.random(d.nseq).astype(np.float32)))
        d.step()
        torch.cuda.synchronize()
        for s in range(d.nseq):
            d.check_rows(f"step {n}, sequence {s}", d.step_buffers[1][s:s + 1].double().cpu(), ids[s], [len(ids[s]) - 1])
        d.check_draw(f"step {n}")


@pytest.mark.parametrize("m", range(len(MODELS)))
def test_a_captured_step_replays_as_the_eager_one(m):
    """The step's append, attention and draw as one graph: every replay gives
    the bits of the eager step, with eager work on the same buffers between."""
    results = []
    for captured in (False, True):
        d = Decoder(200 + m, **MODELS[m], **DRAWS)
        rng = np.random.default_rng(50 + m)
        d.read_prompt()
        d.u.copy_(torch.from_numpy(rng.random(d.nseq).astype(np.float32)))
        d.read_questions()
        lens, tokens = d.lens.clone(), d.tokens.clone()
        run = d.step
        if captured:
            side = torch.cuda.Stream()  # the libraries' first calls, outside the capture
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                d.step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                d.step()
            d.lens.copy_(lens)
            d.tokens.copy_(tokens)
            run = graph.replay
        steps = []
        for _ in range(STEPS):
            d.u.copy_(torch.from_numpy(rng.random(d.nseq).astype(np.float32)))
            run()
            torch.cuda.synchronize()
            d.check_draw("step")
            steps.append((d.step_buffers[1].clone(), d.tokens.clone(), d.logprob.clone(), d.lens.clone()))
        results.append(steps)
    for eager, replayed in zip(*results):
        for a, b in zip(eager, replayed):
            assert torch.equal(a, b)
