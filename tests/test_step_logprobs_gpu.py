"""GPU parity of token_logprobs with the float64 oracle.

Token ids must be equal. Tolerances: a thread adds at most n = 32 ceil(V / 8192) positive terms one
after another, then about 16 levels of a tree, each term off by at most 2^-22 + |t| 2^-22 (the
exponential and its argument, t = x - m): relative to S at most (n + 16) 2^-24 + (1 + E|t|) 2^-22, where E is
the mean under p; log S is off by as much, A / S by as much times 2 E|t|, and every result by two roundings
of its size (2^-23).
"""
import numpy as np
import pytest
import torch

from fast_v2_amd import ops
from oracle import paged_step as ps

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _check(logits, tokens, top_k, what=""):
    """``logits`` [..., V] on the GPU; tokens None, [...] or [..., M]."""
    V = logits.shape[-1]
    got = ops.token_logprobs(logits, tokens, top_k)
    x = logits.double().cpu().numpy().reshape(-1, V)
    n_rows = x.shape[0]
    t = None if tokens is None else tokens.cpu().numpy().reshape(n_rows, -1)
    lp, ent, top, ids = ps.token_logprobs_np(x, t, top_k)
    with np.errstate(invalid="ignore"):
        m = x.max(-1, keepdims=True)
        p = np.where(x > -np.inf, np.exp(x - m), 0.0)
        mean = (p * np.where(p > 0, m - x, 0.0)).sum(-1) / p.sum(-1)
    s_off = (32 * -(-V // 8192) + 16) * 2 ** -24 + (1 + np.nan_to_num(mean)) * 2 ** -22
    for name, a, b, tol in (("entropy", got.entropy, ent, s_off * (1 + 2 * np.nan_to_num(mean))),
                            ("logprobs", got.logprobs, lp, s_off[:, None]),
                            ("top_logprobs", got.top_logprobs, top, s_off[:, None])):
        if a is None:
            continue
        assert a.dtype == F32 and a.shape[:logits.dim() - 1] == logits.shape[:-1]
        a = a.double().cpu().numpy().reshape(b.shape)
        fine = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~fine & ~np.isnan(b)], b[~fine & ~np.isnan(b)]), (what, name)
        err = np.abs(np.where(fine, a, 0) - np.where(fine, b, 0))
        tol = tol + np.abs(np.where(fine, b, 0)) * 2 ** -23
        assert (err <= tol).all(), (what, name, (err - tol).max())
    if top_k:
        assert got.top_tokens.dtype == torch.int64
        assert np.array_equal(got.top_tokens.cpu().numpy().reshape(ids.shape), ids), (what, "ids")
    return got


def _randn(gpu, shape, dtype, seed, scale=2.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(gpu)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [1, 2, 7, 33, 256, 1000, 2048, 2049, 8191, 8192, 8200, 32001, 152064])
def test_vocabularies(gpu, V, dtype):
    print(f"case logprobs V={V} {dtype}", flush=True)
    x = _randn(gpu, (5, V), dtype, V)
    g = torch.Generator(device="cpu").manual_seed(1)
    tokens = torch.randint(0, V, (5, 3), generator=g).to(gpu)
    for k in (0, 1, 5, 20, 32):
        if k <= V:
            _check(x, tokens, k, (V, k))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,V", [(1, 152064), (130, 20001), (700, 9000), (2100, 9000), (2500, 100), (4000, 5)])
def test_row_counts(gpu, rows, V, dtype):
    """Rows shared by workgroups, and workgroups of a whole row of several steps."""
    print(f"case logprobs {rows}x{V} {dtype}", flush=True)
    x = _randn(gpu, (rows, V), dtype, rows)
    _check(x, torch.arange(rows, device=gpu) % V, min(V, 8))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,V", [(1, 16384), (1, 16385), (2, 16392), (5, 24571), (447, 20001), (448, 20001), (447, 33001),
                                    (640, 33001)])
def test_shared_and_whole_rows(gpu, rows, V, dtype):
    """On either side of the rule by which workgroups share rows; every second row starts inside a vector."""
    print(f"case logprobs shared {rows}x{V} {dtype}", flush=True)
    x = _randn(gpu, (rows, V + 1), dtype, rows + V)[:, 1:]
    tokens = torch.arange(3 * rows, device=gpu).view(rows, 3) * 1001 % V
    _check(x, tokens, 20, (rows, V))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [20011, 152064])
def test_orders_of_shared_rows(gpu, V, dtype):
    print(f"case logprobs orders V={V} {dtype}", flush=True)
    at = torch.arange(V, device=gpu)
    up = at.float() * (60.0 / V)
    x = torch.stack([up, up.flip(0), torch.zeros_like(up), (at % 7).float(), torch.where(at == V - 3, 9.0, 1.0), up.round(),
                     -up * 100, torch.where(at % 1000 == 999, 5.0, -float("inf"))])
    for k in (1, 20, 32):
        _check(x.to(dtype), torch.full((len(x),), 999, device=gpu), k, (V, dtype, k))


@pytest.mark.parametrize("rows", [3, 2200])
def test_orders(gpu, rows):
    """Ties, sorted and constant rows: the alternatives' worst cases."""
    V = 6007
    up = torch.arange(V, device=gpu).float() * 0.01
    base = [up, up.flip(0), torch.zeros(V, device=gpu), (torch.arange(V, device=gpu) % 7).float(),
            torch.where(torch.arange(V, device=gpu) == 4001, 9.0, 1.0), (up * 10).round(), -up * 100]
    x = torch.stack([base[r % len(base)] for r in range(rows if rows < 100 else 21)])
    if rows > 100:
        x = x.repeat(rows // 21 + 1, 1)[:rows]
    for dtype in (BF16, F16, F32):
        for k in (1, 2, 20, 32):
            print(f"case logprobs orders rows={rows} {dtype} k={k}", flush=True)
            _check(x.to(dtype), torch.zeros(len(x), dtype=torch.int64, device=gpu), k, (dtype, k))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,V", [(12, 9001), (2400, 700), (12, 152064)])
def test_excluded_and_bad_logits(gpu, rows, V, dtype):
    print(f"case logprobs bad {rows}x{V} {dtype}", flush=True)
    x = _randn(gpu, (rows, V), dtype, 5)
    low = torch.finfo(dtype).min
    x[0, 1::2] = -float("inf")
    x[1] = -float("inf")                      # nothing left
    x[2] = -float("inf")
    x[2, [5, 600]] = torch.tensor([1.0, 2.0], dtype=dtype, device=gpu)  # two words left
    x[3, 77] = float("nan")
    x[4, V - 1] = float("inf")
    x[5] = low                                # masks of the type's lowest value
    x[6] = low
    x[6, 300] = 3.0
    x[7] = torch.finfo(dtype).max
    x[8, 0] = -float("inf")
    x[9] = -float("inf")
    x[9, V - 1] = low                         # one word of the lowest value left
    x[10, :] = float("nan")
    x[11, ::3], x[11, 1::3] = low, -float("inf")
    tokens = torch.tensor([[0, 1, -1, V, V - 1, 2 ** 40]], device=gpu).repeat(rows, 1)
    for k in (0, 3, 32):
        got = _check(x, tokens, k, (rows, V, dtype, k))
        assert got.logprobs[1].isnan().all() and got.entropy[[1, 3, 4, 10]].isnan().all()
        assert not got.entropy[[0, 2, 5, 6, 7, 8, 9, 11]].isnan().any()


def test_shapes_and_strides(gpu):
    V = 1003
    x = _randn(gpu, (3, 9, V), BF16, 6)
    tok = torch.randint(0, V, (3, 9), generator=torch.Generator().manual_seed(2)).to(gpu)
    shifted = _check(x[:, :-1], tok[:, 1:], 4)          # a text's logits score the tokens after them
    # copied rows start at other offsets from 16 bytes, so other threads add their terms: twice the
    # bound of one form, 2 (48 x 2^-24 + 13 x 2^-22) with E|t| <= 12, and the roundings 2 x 16 x 2^-23
    copied = ops.token_logprobs(x[:, :-1].contiguous(), tok[:, 1:].contiguous()).logprobs
    torch.testing.assert_close(shifted.logprobs, copied, atol=1.6e-5, rtol=0)
    _check(x[1:, ::2], tok[1:, ::2, None], 2)
    _check(x[..., 1:900], tok[..., None].clamp(max=898), 3)   # rows off 16 bytes, others' logits around
    _check(x.permute(2, 0, 1).contiguous().permute(1, 2, 0), tok, 3)
    _check(x[0, 0], tok[0, 0], 3)                        # one row
    _check(x.view(1, 3, 9, V), tok.view(1, 3, 9), 3)
    _check(x.view(3, 3, 3, V)[:, 1:], tok.view(3, 3, 3)[:, 1:].int(), 3)
    _check(x[:, :1].expand(-1, 4, -1), None, 3)
    assert ops.token_logprobs(x).logprobs is None
    for shape in ((0, V), (2, 0, V)):
        got = ops.token_logprobs(x.new_zeros(shape), torch.zeros(shape[:-1], dtype=torch.int64, device=gpu), 2)
        assert got.logprobs.shape == shape[:-1] and got.top_tokens.shape == (*shape[:-1], 2)
    assert ops.token_logprobs(x, torch.zeros(3, 9, 0, dtype=torch.int64, device=gpu)).logprobs.shape == (3, 9, 0)


def test_rows_past_32_bits(gpu):
    """The last rows of logits that do not fit 2^32 bytes."""
    V, rows = 152064, 14200
    x = torch.zeros(rows, V, dtype=BF16, device=gpu)
    x[-2:] = _randn(gpu, (2, V), BF16, 8)
    got = ops.token_logprobs(x, torch.arange(rows, device=gpu), 3)
    want = _check(x[-2:].clone(), torch.arange(rows - 2, rows, device=gpu), 3)
    assert torch.equal(got.top_tokens[-2:], want.top_tokens)
    torch.testing.assert_close(got.logprobs[-2:], want.logprobs, atol=1e-4, rtol=0)
    assert got.top_tokens[:-2].eq(torch.arange(3, device=gpu)).all()


def test_captured_and_overlapping(gpu):
    """Two graphs captured on one stream, replayed on two streams at once, with eager calls beside them."""
    V = 40000
    xs = [_randn(gpu, (6, V), BF16, 10 + i) for i in range(2)]
    tok = torch.arange(6, device=gpu)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        ops.token_logprobs(xs[0], tok, 5)
        for x in xs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(ops.token_logprobs(x, tok, 5))
            graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(4):
        for x in xs:
            x.normal_(std=step + 1)
        torch.cuda.synchronize()
        for _ in range(10):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            ops.token_logprobs(xs[0], tok, 5)
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            want = ops.token_logprobs(x, tok, 5)
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_refusals(gpu):
    x = torch.zeros(2, 10, dtype=BF16, device=gpu)
    tok = torch.zeros(2, dtype=torch.int64, device=gpu)
    for args in ((x.double(), tok, 1), (x.long(), tok, 1), (x, tok.float(), 1), (x, tok[:1], 1), (x, tok, 11), (x, tok, -1),
                 (torch.zeros(2, 50, dtype=BF16, device=gpu), tok, 33), (x, tok.cpu(), 1), (x[:, :0], tok, 0)):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(*args)
    with pytest.raises(RuntimeError, match="backward"):
        ops.token_logprobs(x.float().requires_grad_(), tok)
