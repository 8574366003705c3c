"""The paged cache's operators and the log probabilities together, as a serving
loop uses them: packed prompts, parallel samples forked from one of them, a
rejected token, a finished sample, compaction, all through the trait's other
ops.  Every step's logits are held to the same model on the flat cache
(kv_write / attention in the reference's order), sequence by sequence, by the bar
the reference sets for a non-oracle backend: within 1e-3, and the same argmax
(tests/backends.rs:129-148)."""
import numpy as np
import pytest

import kernrt_b200
from kernrt_b200 import BF16, F32

pytestmark = pytest.mark.gpu

LAYERS, DIM, HEADS, KV_HEADS, HEAD, HIDDEN, VOCAB, THETA, EPS = 2, 256, 4, 2, 64, 512, 1000, 1e4, 1e-5
Q, KV = HEADS * HEAD, KV_HEADS * HEAD


class Model:
    """The weights on one backend, and a forward pass over packed rows."""

    def __init__(self, b):
        self.b = b
        rng = np.random.default_rng(0)

        def mat(o, i):
            return b.prepare_matrix(F32, (rng.standard_normal((o, i)) / np.sqrt(i)).astype(np.float32), None, o, i)

        def norm():
            return b.upload((1 + 0.1 * rng.standard_normal(DIM)).astype(np.float32))

        b.prepare_embedding(F32, rng.standard_normal((VOCAB, DIM)).astype(np.float32), None, VOCAB, DIM)
        self.layers = [dict(att=norm(), q=mat(Q, DIM), k=mat(KV, DIM), v=mat(KV, DIM), o=mat(DIM, Q), ffn=norm(),
                            gate=mat(HIDDEN, DIM), up=mat(HIDDEN, DIM), down=mat(DIM, HIDDEN)) for _ in range(LAYERS)]
        self.final, self.out = norm(), mat(VOCAB, DIM)

    def forward(self, tokens, positions, attend):
        """attend(layer, q, k, v, out) is the cache's part.  Returns the logits' buffer."""
        b, n = self.b, len(tokens)
        x, xb, q, k, v, o, g, u = (b.alloc(n * w) for w in (DIM, DIM, Q, KV, KV, Q, HIDDEN, HIDDEN))
        logits = b.alloc(n * VOCAB)
        for i, t in enumerate(tokens):
            b.embed(int(t), x, i * DIM)
        for layer, w in enumerate(self.layers):
            b.rms_norm(xb, x, w["att"], n, DIM, EPS)
            b.project_qkv(w["q"], w["k"], w["v"], xb, q, k, v, n)
            b.rope(q, k, Q, KV, n, positions, HEAD, THETA, False)
            attend(layer, q, k, v, o)
            b.project(w["o"], o, xb, n)
            b.add_in_place(x, xb, n * DIM)
            b.rms_norm(xb, x, w["ffn"], n, DIM, EPS)
            b.project_gate_up(w["gate"], w["up"], xb, g, u, n)
            b.silu_mul(g, u, n * HIDDEN)
            b.project(w["down"], g, xb, n)
            b.add_in_place(x, xb, n * DIM)
        b.rms_norm(xb, x, self.final, n, DIM, EPS)
        b.project(self.out, xb, logits, n)
        for h in (x, xb, q, k, v, o, g, u):
            b.free(h)
        return logits


def flat_logits(model, tokens):
    """The logits of every position of one sequence on the flat cache."""
    b, n = model.b, len(tokens)
    b.kv_prepare(LAYERS, KV, 128)
    att = b.alloc(n * HEADS * 128)

    def attend(layer, q, k, v, o):
        b.kv_write(layer, np.arange(n), k, v, n)
        b.attention(q, o, att, layer, [(0, i, 0, 0) for i in range(n)], HEADS, HEADS // KV_HEADS, HEAD, KV, 128)

    h = model.forward(tokens, np.arange(n), attend)
    out = b.read(h, n * VOCAB).reshape(n, VOCAB)
    b.free(h)
    b.free(att)
    return out


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_serving_loop(kind):
    rng = np.random.default_rng(1)
    bar = 1e-3 if kind == F32 else 5e-2  # bf16 keys and values: the bar of a rounded format (tests/backends.rs:389-426)
    with kernrt_b200.CudaBackend(0) as b, kernrt_b200.CudaBackend(0) as flat:
        model, plain = Model(b), Model(flat)
        p = b.pages_create(kind, LAYERS, HEADS, KV_HEADS, HEAD, 16, 24, 8, 100)
        texts = {}

        def step(seqs, more):
            """seqs[i] takes the tokens more[i]; checks and returns the logits."""
            rows = [len(m) for m in more]
            b.pages_step(p, seqs, rows)
            tokens, positions, want = [], [], []
            for s, m in zip(seqs, more):
                at = len(texts[s])
                texts[s] = texts[s] + [int(t) for t in m]
                tokens += [int(t) for t in m]
                positions += range(at, at + len(m))
                want.append(flat_logits(plain, texts[s])[at:])

            def attend(layer, q, k, v, o):
                b.pages_write(p, layer, k, v)
                b.pages_attention(p, layer, q, o)

            h = model.forward(tokens, positions, attend)
            n = len(tokens)
            got = b.read(h, n * VOCAB).reshape(n, VOCAB)
            want = np.concatenate(want)
            assert np.abs(got - want).max() <= bar
            top2 = np.sort(want, axis=1)[:, -2:]
            clear = top2[:, 1] - top2[:, 0] > 2 * bar
            assert (got.argmax(1) == want.argmax(1))[clear].all() and clear.any()
            # the log probability of each row's next token, and the alternatives
            nxt = rng.integers(0, VOCAB, n).astype(np.int32)
            hs = [b.upload_bytes(nxt), b.alloc(n), b.alloc(n), b.alloc_bytes(4 * n * 5), b.alloc(n * 5)]
            b.logprobs(h, n, VOCAB, hs[0], hs[1], hs[2], 5, hs[3], hs[4])
            lp, ent = b.read(hs[1], n), b.read(hs[2], n)
            ids, tops = b.read_bytes(hs[3], 4 * n * 5, np.int32).reshape(n, 5), b.read(hs[4], n * 5).reshape(n, 5)
            x = got.astype(np.float64)
            logp = x - x.max(1, keepdims=True)
            logp -= np.log(np.exp(logp).sum(1, keepdims=True))
            assert np.allclose(lp, logp[np.arange(n), nxt], rtol=2.0 ** -22, atol=2.0 ** -14)
            assert np.allclose(ent, -(np.exp(logp) * logp).sum(1), atol=2.0 ** -13)
            order = np.argsort(-x, axis=1, kind="stable")[:, :5]
            assert np.array_equal(ids, order)
            assert np.allclose(tops, np.take_along_axis(logp, order, 1), rtol=2.0 ** -22, atol=2.0 ** -14)
            for buf in hs + [h]:
                b.free(buf)
            return got

        def draw(n):
            return rng.integers(0, VOCAB, n).tolist()

        one, two = b.seq_open(p), b.seq_open(p)
        texts[one] = texts[two] = []
        step([one, two], [draw(37), draw(5)])          # two prompts, packed
        kids = b.seq_fork(p, one, 37, 3)               # three samples of the first
        for k in kids:
            texts[k] = texts[one]
        for _ in range(3):
            step(kids + [two], [draw(1) for _ in range(4)])
        b.seq_trim(p, kids[1], 38)                     # two tokens rejected
        texts[kids[1]] = texts[kids[1]][:38]
        b.seq_close(p, [kids[0], one])                 # a sample ends; the prompt goes on in the others
        b.pages_compact(p)
        step([two, kids[2], kids[1]], [draw(20), draw(1), draw(4)])  # a chunk, a token, drafts
        copy = b.seq_copy(p, two, 18)
        texts[copy] = texts[two][:18]
        step([copy, two, kids[1]], [draw(2), draw(1), draw(1)])
        b.seq_close(p, [two, copy] + kids[1:])
        assert b.pages_ptr(p).available == 24
        b.pages_destroy(p)
