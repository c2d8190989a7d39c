"""GPU: whole serving steps over a paged cache: the token list, the row norm, the projections, rotary
positions into the pages, the attention, and the log probabilities of the logits, on one stream
with nothing waited for in between.  Each operator's output is held against numpy in 64 bits on the inputs that it
had; the same steps captured into a graph and replayed give the same bits."""
import numpy as np
import pytest

from tests import paged_ref
from tests import serving_ref as ref
from tests.helpers import assert_close, rng, say

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, HQ, HKV, D, VOCAB, PAGE, WIDTH, ROWS, TOP = 128, 256, 4, 2, 64, 1024, 16, 12, 6, 5
QKV = (HQ + 2 * HKV) * D
# (tokens asked for, granted) of each row, step by step: pieces of prompts, then some and single tokens, then single ones
STEPS = [([60, 7, 0, 33, 1, 16], [1, 1, 1, 1, 1, 1]), ([40, 1, 5, 1, 1, 70], [1, 1, 1, 0, 1, 1]),
         ([1, 1, 1, 1, 1, 1], [1, 1, 1, 1, 0, 1])]


class Step:
    def __init__(self, hip, cache):
        r = rng(77)
        self.hip, self.cache = hip, cache
        bf16 = lambda *shape, scale=1.0: ref.rounded(r.normal(size=shape).astype(np.float32) * scale, "bf16")   # noqa: E731
        self.num = ROWS * WIDTH + 2
        self.tables = r.permutation(self.num)[:ROWS * WIDTH].astype(np.int32).reshape(ROWS, WIDTH)
        self.turns = ref.turns("none", D, 10000.0)
        self.wqkv, self.wo = bf16(QKV, HIDDEN, scale=HIDDEN ** -0.5), bf16(HIDDEN, HQ * D, scale=HIDDEN ** -0.5)
        self.head, _ = ref.cpuref.e4m3_encode(r.normal(size=(VOCAB, HIDDEN)).astype(np.float32), 0.01), None
        self.norm1, self.norm2 = bf16(HIDDEN), bf16(HIDDEN)
        self.scales = (0.02, 0.03) if cache == "fp8" else (1.0, 1.0)
        self.targets = r.integers(0, VOCAB, TOKENS).astype(np.int32)
        self.inputs = [(bf16(TOKENS, HIDDEN), bf16(TOKENS, HIDDEN)) for _ in STEPS]
        up = hip.DeviceBuffer.from_array
        self.w = [up(x) for x in (self.wqkv[0], self.wo[0], self.head, self.norm1[0], self.norm2[0], self.turns, self.targets, self.tables)]
        es = 1 if cache == "fp8" else 2
        self.stride = HKV * PAGE * D
        self.pools = [hip.DeviceBuffer(self.num * self.stride * es) for _ in "kv"]
        sizes = dict(lengths=4 * ROWS, need=4 * ROWS, granted=4 * ROWS, starts=4 * ROWS + 4, rows=4 * TOKENS, positions=4 * TOKENS,
                     now=4 * ROWS, x=2 * TOKENS * HIDDEN, res=2 * TOKENS * HIDDEN, sum=2 * TOKENS * HIDDEN, y=2 * TOKENS * HIDDEN,
                     qkv=2 * TOKENS * QKV, q=2 * TOKENS * HQ * D, att=2 * TOKENS * HQ * D, h=2 * TOKENS * HIDDEN,
                     sum2=2 * TOKENS * HIDDEN, y8=TOKENS * HIDDEN, logits=4 * TOKENS * VOCAB, logp=4 * TOKENS, entropy=4 * TOKENS,
                     tlp=4 * TOKENS * TOP, ids=4 * TOKENS * TOP,
                     ws=hip.paged_attn_chunk_workspace(ROWS, TOKENS, HQ, HKV, D), lws=hip.logprobs_workspace(TOKENS, VOCAB, TOP))
        self.b = {k: hip.DeviceBuffer(max(n, 16)) for k, n in sizes.items()}

    def reset(self):
        for p in self.pools + list(self.b.values()):
            p.fill_bytes(0x5A)
        self.b["now"].upload(np.array([0, 20, 3, 0, 100, 50], np.int32))
        # the tokens that were there before: anything finite
        r = rng(78)
        for p in self.pools:
            if self.cache == "fp8":
                p.upload(r.integers(0, 0x60, self.num * self.stride).astype(np.uint8))
            else:
                p.upload(ref.rounded(r.normal(size=self.num * self.stride).astype(np.float32), "bf16")[0])

    def feed(self, i):
        b = self.b
        b["att"].fill_bytes(0x5A)
        self.old = b["now"].download(np.int32, (ROWS,))
        b["lengths"].upload(self.old)
        b["need"].upload(np.array(STEPS[i][0], np.int32))
        b["granted"].upload(np.array(STEPS[i][1], np.int32))
        b["x"].upload(self.inputs[i][0][0])
        b["res"].upload(self.inputs[i][1][0])

    def run(self, st):
        h, b = self.hip, {k: v.ptr for k, v in self.b.items()}
        wqkv, wo, head, n1, n2, turns, targets, tables = (x.ptr for x in self.w)
        k, v = (p.ptr for p in self.pools)
        cache = h.F8E4M3 if self.cache == "fp8" else h.BF16
        h.kv_slots(ROWS, b["lengths"], b["need"], b["granted"], TOKENS, b["starts"], b["rows"], b["positions"], b["now"], st)
        h.rmsnorm_rows(h.BF16, h.BF16, TOKENS, HIDDEN, b["x"], HIDDEN, b["res"], HIDDEN, b["sum"], HIDDEN, n1, 1e-5, b["y"], HIDDEN,
                       stream=st)
        h.gemm(h.BF16, h.BF16, h.BF16, TOKENS, QKV, HIDDEN, b["y"], HIDDEN, h.ROW_MAJOR, wqkv, HIDDEN, h.COL_MAJOR, b["qkv"], QKV,
               1.0, 1.0, 0, st)
        h.rope_append(h.BF16, cache, h.ROPE_HALF, TOKENS, HQ, HKV, D, D, b["qkv"], QKV, b["q"], HQ * D, b["qkv"] + 2 * HQ * D, QKV,
                      b["qkv"] + 2 * (HQ + HKV) * D, QKV, b["rows"], b["positions"], turns, 1.0, k, v, self.num, PAGE, self.stride,
                      tables, ROWS, WIDTH, *self.scales, stream=st)
        h.paged_attn_chunk(h.BF16, cache, ROWS, TOKENS, HQ, HKV, D, b["q"], HQ * D, b["starts"], k, v, self.num, PAGE, self.stride,
                           tables, WIDTH, b["now"], b["att"], HQ * D, D ** -0.5, *self.scales, workspace=b["ws"],
                           workspace_bytes=self.b["ws"].nbytes, stream=st)
        h.gemm(h.BF16, h.BF16, h.BF16, TOKENS, HIDDEN, HQ * D, b["att"], HQ * D, h.ROW_MAJOR, wo, HQ * D, h.COL_MAJOR, b["h"], HIDDEN,
               1.0, 1.0, 0, st)
        h.rmsnorm_rows(h.BF16, h.F8E4M3, TOKENS, HIDDEN, b["h"], HIDDEN, b["sum"], HIDDEN, b["sum2"], HIDDEN, n2, 1e-5, b["y8"], HIDDEN,
                       scale=0.02, stream=st)
        h.gemm(h.F8E4M3, h.F8E4M3, h.F32, TOKENS, VOCAB, HIDDEN, b["y8"], HIDDEN, h.ROW_MAJOR, head, HIDDEN, h.COL_MAJOR, b["logits"],
               VOCAB, 0.02, 0.01, 0, st)
        h.logprobs_rows(h.F32, TOKENS, VOCAB, b["logits"], VOCAB, 0.7, targets, b["logp"], b["entropy"], TOP, b["tlp"], b["ids"],
                        b["lws"], self.b["lws"].nbytes, st)

    def outputs(self):
        """The step's buffers; of the tokens behind the list what no operator leaves as it was is not compared."""
        shapes = dict(starts=(np.int32, (ROWS + 1,)), rows=(np.int32, (TOKENS,)), positions=(np.int32, (TOKENS,)), now=(np.int32, (ROWS,)),
                      sum=(np.uint16, (TOKENS, HIDDEN)), y=(np.uint16, (TOKENS, HIDDEN)), qkv=(np.uint16, (TOKENS, QKV)),
                      q=(np.uint16, (TOKENS, HQ * D)), att=(np.uint16, (TOKENS, HQ * D)), h=(np.uint16, (TOKENS, HIDDEN)),
                      sum2=(np.uint16, (TOKENS, HIDDEN)), y8=(np.uint8, (TOKENS, HIDDEN)), logits=(np.uint32, (TOKENS, VOCAB)),
                      logp=(np.uint32, (TOKENS,)), entropy=(np.uint32, (TOKENS,)), tlp=(np.uint32, (TOKENS, TOP)), ids=(np.int32, (TOKENS, TOP)))
        out = {k: self.b[k].download(*s) for k, s in shapes.items()}
        out["pools"] = [p.download(np.uint8, (p.nbytes,)) for p in self.pools]
        return out

    def check(self, i, out, before):
        need, granted = STEPS[i]
        for name, want in zip(("starts", "rows", "positions", "now"), ref.slots(self.old.tolist(), need, granted, TOKENS)):
            assert np.array_equal(out[name], want), name
        n = int(out["starts"][-1])
        rows, positions = out["rows"][:n], out["positions"][:n]
        bf = lambda x: ref.values(x[:n], "bf16")   # noqa: E731
        # the first norm
        s, y, e = ref.rmsnorm(self.inputs[i][0][1][:n], self.inputs[i][1][1][:n], self.norm1[1], 1e-5)
        ref.within(bf(out["sum"]), s, np.abs(s) * ref.EPS, "bf16", "sum")
        ref.within(bf(out["y"]), y, np.abs(y) * e, "bf16", "norm")
        assert_close(bf(out["qkv"]), bf(out["y"]) @ self.wqkv[1].T, atol=2e-2, rtol=1e-2, what="projection")
        # rotary positions, and the pages
        x = bf(out["qkv"]).reshape(n, HQ + 2 * HKV, D)
        want, err = ref.rope(x[:, :HQ + HKV], positions, self.turns, 1.0, "half")
        q = bf(out["q"]).reshape(n, HQ, D)
        ref.within(q, want[:, :HQ], err[:, :HQ], "bf16", "q")
        page, slot = self.tables[rows, positions // PAGE], positions % PAGE
        stored = []
        for name, new, err, was, now, scale in (("k", want[:, HQ:], err[:, HQ:], before[0], out["pools"][0], self.scales[0]),
                                                ("v", x[:, HQ + HKV:].astype(np.float64), 0.0, before[1], out["pools"][1], self.scales[1])):
            kind = "fp8" if self.cache == "fp8" else "bf16"
            now, was = (p.view(ref.NP[kind]).reshape(self.num, HKV, PAGE, D).copy() for p in (now, was))
            err = (err + np.abs(new) * 2 * ref.EPS * (kind == "fp8")) / scale
            ref.within(ref.values(now[page, :, slot], kind), new / scale, err, kind, name)
            stored.append(ref.values(now, kind).astype(np.float64) * scale)
            now[page, :, slot] = was[page, :, slot]
            assert np.array_equal(now, was), "wrote elsewhere in the pages"
        # the attention
        att = bf(out["att"]).reshape(n, HQ, D).astype(np.float64)
        for t in range(n):
            at = np.arange(positions[t] + 1)
            ids = self.tables[rows[t], at // PAGE]
            for head in range(HQ):
                kk, vv = (p[ids, head // (HQ // HKV), at % PAGE] for p in stored)
                want, spread, size = paged_ref.attention(q[t, head], kk, vv, D ** -0.5)
                bound = paged_ref.error_bound(want, spread, size, "bf16", D, len(at), 2.0 ** -8)
                assert (np.abs(att[t, head] - want) <= bound).all(), ("attention", t, head)
        assert (out["att"][n:] == 0x5A5A).all(), "rows behind the list"
        assert_close(bf(out["h"]), bf(out["att"]) @ self.wo[1].T, atol=2e-2, rtol=1e-2, what="output projection")
        # the second norm, into codes of a given scale
        s, y, e = ref.rmsnorm(bf(out["h"]), bf(out["sum"]), self.norm2[1], 1e-5)
        ref.within(bf(out["sum2"]), s, np.abs(s) * ref.EPS, "bf16", "sum 2")
        ref.within(ref.values(out["y8"][:n], "fp8"), y / 0.02, np.abs(y / 0.02) * (2 * e + 4 * ref.EPS), "fp8", "norm 2")
        logits = out["logits"].view(np.float32)[:n]
        assert_close(logits, (ref.values(out["y8"][:n], "fp8") @ ref.values(self.head, "fp8").T) * np.float32(0.0002), atol=2e-2, rtol=1e-2,
                     what="logits")
        logp, entropy, tlp, ids, e, e_entropy = ref.logprobs(logits, np.float32(0.7), self.targets[:n], TOP)
        assert np.array_equal(out["ids"][:n], ids), "top columns"
        f = lambda x: x.view(np.float32)[:n]   # noqa: E731
        ref.within(f(out["logp"])[:, None], logp[:, None], e(logp[:, None]), "f32", "logp")
        ref.within(f(out["tlp"]), tlp, e(tlp), "f32", "top")
        ref.within(f(out["entropy"]), entropy, e_entropy, "f32", "entropy")
        return n


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_serving_steps(hip, cache):
    step, st, other = Step(hip, cache), hip.Stream(), hip.Stream()
    step.reset()
    eager = []
    for i in range(len(STEPS)):
        say(f"serving step {i}, {cache} cache")
        step.feed(i)
        before = [p.download(np.uint8, (p.nbytes,)) for p in step.pools]
        hip.synchronize()
        step.run(st)
        st.synchronize()
        eager.append(step.outputs())
        eager[-1]["n"] = step.check(i, eager[-1], before)
    say("captured")
    beside = Step(hip, cache)   # eager work of the same operators on another stream, between and beside the replays
    beside.reset()
    with hip.Graph(st) as graph:
        step.run(st)
    for turn in range(2):
        step.reset()
        for i in range(len(STEPS)):
            step.feed(i)
            beside.feed(0)
            hip.synchronize()
            graph.launch()
            beside.run(other)
            st.synchronize()
            other.synchronize()
            got, want = step.outputs(), eager[i]
            say(f"replay {turn} of step {i}")
            for name, x in got.items():
                if name == "pools":
                    assert all(np.array_equal(a, b) for a, b in zip(x, want[name])), (turn, i, name)
                else:
                    n = want["n"] if len(x) == TOKENS else len(x)
                    assert np.array_equal(x[:n], want[name][:n]), (turn, i, name)
    graph.close()
    st.close()
    other.close()
