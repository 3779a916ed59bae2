"""A paged step as a server makes it, from the requests' lengths to the scores: pages and slots,
head norms + rotation + the paged write, block attention over the pages, lm_head, log
probabilities, and the rejected part of a draft given back."""
import numpy as np
import pytest
import torch

from fast_v2_amd import _ffi, ops
from oracle import attention as oa
from oracle import paged_step as ps

pytestmark = pytest.mark.gpu

B, W, Hq, Hkv, D, PAGE, MOST, V = 5, 8, 6, 2, 128, 32, 6, 1000


class _Server:
    def __init__(self, gpu, head_major):
        g = torch.Generator(device="cpu").manual_seed(11)
        self.free = torch.randperm(B * MOST, generator=g).int().to(gpu)
        self.count = torch.tensor([B * MOST], dtype=torch.int32, device=gpu)
        self.lens = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.table = torch.zeros(B, MOST, dtype=torch.int32, device=gpu)
        shape = (B * MOST, Hkv, PAGE, D) if head_major else (B * MOST, PAGE, Hkv, D)
        self.kc, self.vc = (torch.zeros(shape, dtype=torch.bfloat16, device=gpu) for _ in range(2))
        if head_major:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        self.freq, self.scale = ops.rope_frequencies(D, 1e6, "yarn", 4.0, device=gpu)
        self.w = (torch.rand(2, D, generator=g) + 0.5).bfloat16().to(gpu)
        self.head = (torch.randn(V, Hq * D, generator=g) * 0.05).bfloat16().to(gpu)
        self.new = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.x = torch.zeros(B, W, Hq + 2 * Hkv, D, dtype=torch.bfloat16, device=gpu)
        self.tokens = torch.zeros(B, W, dtype=torch.int64, device=gpu)
        self.keep = torch.zeros(B, dtype=torch.int32, device=gpu)

    def pool(self):
        return self.lens, self.table, self.free, self.count, PAGE

    def step(self):
        rows = ops.assign_pages(self.new, *self.pool(), width=W)
        q = ops.norm_rope_kv_write(self.x[:, :, :Hq], self.x[:, :, Hq:Hq + Hkv], self.x[:, :, Hq + Hkv:], rows.positions,
                                   self.freq, self.w[0], self.w[1], 1e-6, self.kc, self.vc, rows.slots,
                                   rope_scale=self.scale)
        att = ops.block_attn(q, self.kc, self.vc, rows.seqlens, mask_mode=_ffi.MASK_CAUSAL, q_start=rows.starts,
                             page_table=self.table, page_size=PAGE)
        logits = ops.linear(att.view(B, W, Hq * D), self.head)
        scores = ops.token_logprobs(logits, self.tokens, 4)
        ops.release_pages(self.keep, *self.pool())
        return rows, q, att, logits, scores


def _inputs(s, g, step):
    s.new.copy_(torch.randint(1, W + 1, (B,), generator=g))
    s.x.copy_(torch.randn(s.x.shape, generator=g))
    s.tokens.copy_(torch.randint(0, V, (B, W), generator=g))
    s.keep.copy_(torch.randint(0, 8 * (step + 1), (B,), generator=g))


@pytest.mark.parametrize("head_major", [False, True])
def test_steps_against_the_oracles(gpu, head_major):
    s, g = _Server(gpu, head_major), torch.Generator().manual_seed(1)
    lens, free, table = [0] * B, s.free.tolist(), np.zeros((B, MOST), np.int64)
    keys = [np.zeros((0, Hkv, D)) for _ in range(B)]
    vals = [np.zeros((0, Hkv, D)) for _ in range(B)]
    freq, w = s.freq.cpu().double().numpy(), s.w.cpu().double().numpy()
    for step in range(9):
        _inputs(s, g, step)
        new, x = s.new.tolist(), s.x.cpu().double().numpy()
        rows, q, att, logits, scores = s.step()
        want = ps.assign_pages_np(new, lens, table, free, PAGE, width=W)
        assert np.array_equal(rows.slots.cpu().numpy().ravel(), want["slots"])
        pos = want["positions"].reshape(B, W)
        q_want = ps.norm_rope_np(x[:, :, :Hq], pos, freq, w[0], 1e-6, False, s.scale)
        k_want = ps.norm_rope_np(x[:, :, Hq:Hq + Hkv], pos, freq, w[1], 1e-6, False, s.scale)
        for b in range(B):
            n = want["granted"][b]
            assert n == new[b]
            keys[b] = np.concatenate([keys[b], k_want[b, :n]])
            vals[b] = np.concatenate([vals[b], x[b, :n, Hq + Hkv:]])
            for t in range(n):
                # keys up to the token's own, in float64; the kernel's are rounded to bf16, as its output is
                to = want["starts"][b] + t + 1
                k, v = keys[b][:to], vals[b][:to]
                for h in range(Hq):
                    sc = k[:, h // (Hq // Hkv)] @ q_want[b, t, h] * D ** -0.5
                    p = np.exp(sc - sc.max())
                    np.testing.assert_allclose(att[b, t, h].double().cpu().numpy(), p @ v[:, h // (Hq // Hkv)] / p.sum(),
                                               atol=4e-2, rtol=2e-2)
        lg = logits.double().cpu().numpy().reshape(B * W, V)
        lp, ent, top, ids = ps.token_logprobs_np(lg, s.tokens.cpu().numpy().reshape(B * W, 1), 4)
        np.testing.assert_allclose(scores.logprobs.cpu().numpy().ravel(), lp.ravel(), atol=2e-5)
        np.testing.assert_allclose(scores.entropy.cpu().numpy().ravel(), ent, atol=2e-5)
        assert np.array_equal(scores.top_tokens.cpu().numpy().reshape(B * W, 4), ids)
        ps.release_pages_np(s.keep.tolist(), lens, table, free, PAGE)
        for b in range(B):
            keys[b], vals[b] = keys[b][:lens[b]], vals[b][:lens[b]]
        assert s.lens.tolist() == lens and s.free[:len(free)].tolist() == free


def test_the_step_in_a_graph(gpu):
    eager, graphed = _Server(gpu, False), _Server(gpu, False)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphed.step()  # nothing asked for, nothing kept
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = graphed.step()
    torch.cuda.synchronize()
    for step in range(5):
        _inputs(eager, torch.Generator().manual_seed(step), step)
        _inputs(graphed, torch.Generator().manual_seed(step), step)
        want = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        live = want[0].slots >= 0
        assert torch.equal(out[0].slots, want[0].slots) and torch.equal(graphed.table, eager.table)
        for a, b in zip((*out[1:4], *out[4]), (*want[1:4], *want[4])):
            assert torch.equal(a[live], b[live])
        assert torch.equal(graphed.lens, eager.lens) and torch.equal(graphed.count, eager.count)
