"""GPU parity of norm_rope_kv_write with the float64 oracle.

Tolerance: the output's rounding, at most half a step (u = finfo.eps / 2 of |y|; 2^-25 for
fp16 values below its normal range), and the fp32 arithmetic before it: with amp = |x0| + |x1| of the normed pair, the angle's rest of a turn is
off by 2^-25 half turns (2^-23.3 rad) and sin / cos by 2 ulp (2^-23), the norm's mean, rsqrt and two products by at
most 12 x 2^-24, products and sum by 3 x 2^-24: below 2^-19 amp in all.
"""
import numpy as np
import pytest
import torch

from fast_v2_amd import ops
from oracle import paged_step as ps

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _close(got, x, positions, freq, weight, eps, interleaved, scale, what):
    dt = got.dtype
    args = [positions.cpu().numpy(), freq.cpu().double().numpy(),
            None if weight is None else weight.cpu().double().numpy(), eps, interleaved]
    want = ps.norm_rope_np(x.cpu().double().numpy(), *args, scale)
    half = len(freq)
    plain = np.abs(ps.norm_rope_np(x.cpu().double().numpy(), np.zeros_like(args[0]), *args[1:]))
    amp = plain.copy()
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    amp[..., first] = amp[..., second] = (plain[..., first] + plain[..., second]) * scale
    u = torch.finfo(dt).eps / 2
    tol = u * np.abs(want) * (1 + 2 ** -8) + 2 ** -19 * amp + (2 ** -25 if dt == F16 else 0)
    err = np.abs(got.cpu().double().numpy() - want)
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (what, worst, err[worst], tol[worst], want[worst])


def _inputs(gpu, B, S, Hq, Hkv, D, dtype, seed, packed=True):
    g = torch.Generator(device="cpu").manual_seed(seed)
    x = (torch.randn(B, S, Hq + 2 * Hkv, D, generator=g) * 2).to(dtype).to(gpu)
    if packed:
        return x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
    return x[:, :, :Hq].contiguous(), x[:, :, Hq:Hq + Hkv].contiguous(), x[:, :, Hq + Hkv:].contiguous()


def _pools(gpu, pages, page, Hkv, D, dtype, head_major=False):
    out = []
    for fill in (7.0, -3.0):
        shape = (pages, Hkv, page, D) if head_major else (pages, page, Hkv, D)
        t = torch.full(shape, fill, dtype=dtype, device=gpu)
        out.append(t.transpose(1, 2) if head_major else t)
    return out


CASES = [
    # B, S, Hq, Hkv, D, R, interleaved, q norm, k norm, head major
    (1, 1, 28, 4, 128, 128, False, True, True, False),
    (3, 8, 28, 4, 128, 128, False, True, True, True),
    (2, 5, 12, 2, 64, 64, False, True, False, False),
    (2, 5, 12, 2, 64, 32, False, False, True, True),
    (1, 37, 8, 8, 128, 64, False, False, False, False),
    (2, 3, 5, 1, 80, 80, False, True, True, False),    # R / 2 no multiple of 8
    (2, 3, 5, 1, 80, 20, False, True, True, False),
    (2, 3, 5, 1, 80, 2, False, True, True, True),
    (2, 9, 4, 4, 96, 48, True, True, True, False),
    (2, 9, 4, 2, 256, 256, False, True, True, False),
    (1, 2, 64, 64, 256, 66, True, True, True, False),   # more heads than a workgroup holds
    (1, 2, 130, 2, 128, 34, False, True, True, False),
    (1, 4, 3, 1, 8, 8, False, True, True, False),
    (1, 4, 3, 1, 8, 6, True, True, True, False),
    (1, 4, 3, 1, 24, 0, False, True, True, False),      # nothing rotated
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", CASES)
def test_against_float64(gpu, case, dtype):
    B, S, Hq, Hkv, D, R, inter, qn, kn, hm = case
    print(f"case norm_rope {dtype} {case}", flush=True)
    q, k, v = _inputs(gpu, B, S, Hq, Hkv, D, dtype, seed=D + R + S)
    g = torch.Generator(device="cpu").manual_seed(1)
    qw = (torch.rand(D, generator=g) + 0.5).to(dtype).to(gpu) if qn else None
    kw = (torch.rand(D, generator=g) + 0.5).to(dtype).to(gpu) if kn else None
    pos = torch.randint(0, 200000, (B, S), generator=g, dtype=torch.int32).to(gpu)
    freq, scale = ops.rope_frequencies(R, 1e4, "yarn", 4.0)
    page, pages = 16, (B * S) // 16 + 3
    slots = torch.randperm(pages * page, generator=g)[:B * S].view(B, S)
    if B * S > 2:  # rows that have no slot in the pool
        slots.view(-1)[::5] = torch.tensor([-1, pages * page, -2 ** 40, 2 ** 40])[torch.arange(len(slots.view(-1)[::5])) % 4]
    slots = slots.to(gpu)
    kc, vc = _pools(gpu, pages, page, Hkv, D, dtype, hm)
    got, k_got = ops.norm_rope_kv_write(q, k, v, pos, freq.to(gpu), qw, kw, 1e-5, kc, vc, slots, inter, scale, kv_out=True)
    assert got.shape == (B, S, Hq, D) and got.dtype == dtype and got.is_contiguous()
    _close(got, q, pos, freq, qw, 1e-5, inter, scale, "q")
    _close(k_got, k, pos, freq, kw, 1e-5, inter, scale, "k")
    for c, rows, fill in ((kc, k_got, 7.0), (vc, v, -3.0)):
        want = torch.full((pages * page, Hkv, D), fill, dtype=dtype, device=gpu)
        live = (slots >= 0) & (slots < pages * page)
        want[slots[live]] = rows[live]
        assert torch.equal(c.reshape(pages * page, Hkv, D), want)


@pytest.mark.parametrize("heads", [(3, 1, 128, 128, False), (9, 2, 80, 20, False), (2, 2, 64, 64, True), (5, 3, 256, 64, False)])
@pytest.mark.parametrize("B,S", [(1, 600), (3, 427), (1, 1279), (1, 1281), (2, 1279), (1, 2559), (1, 2561), (7, 400)])
def test_token_counts(gpu, B, S, heads):
    """Several workgroups, waves, two waves and one wave to a token, with waves left over."""
    Hq, Hkv, D, R, inter = heads
    test_against_float64(gpu, (B, S, Hq, Hkv, D, R, inter, True, True, False), BF16 if S % 2 else F32)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_far_positions(gpu, dtype):
    """The angles of positions up to the type's end, and negative ones."""
    B, S, H, D = 1, 9, 2, 64
    q, k, v = _inputs(gpu, B, S, H, H, D, dtype, 3)
    pos = torch.tensor([[0, 1, -1, 99999, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31, 123456789]], dtype=torch.int32,
                       device=gpu)
    freq = ops.rope_frequencies(D, 1e4)[0]
    got, k_got = ops.norm_rope_kv_write(q, k, v, pos, freq.to(gpu), kv_out=True)
    _close(got, q, pos, freq, None, 0, False, 1.0, "q")
    _close(k_got, k, pos, freq, None, 0, False, 1.0, "k")


def test_forms_of_the_arguments(gpu):
    """Contiguous and strided, unaligned, 64-bit positions, fp32 and mixed weights: the same result."""
    B, S, Hq, Hkv, D = 2, 7, 6, 2, 64
    q, k, v = _inputs(gpu, B, S, Hq, Hkv, D, BF16, 5)
    pos = torch.arange(B * S, dtype=torch.int32, device=gpu).view(B, S) * 37
    freq = ops.rope_frequencies(D, 1e4)[0].to(gpu)
    w = torch.rand(D, device=gpu).to(BF16)
    want = ops.norm_rope_kv_write(q, k, v, pos, freq, w, w)
    odd = torch.empty(B * S * Hq * D + 1, dtype=BF16, device=gpu)[1:].view(B, S, Hq, D).copy_(q)
    bhsd = q.transpose(1, 2).contiguous().transpose(1, 2)
    last = q.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
    odd_w = torch.empty(D + 1, dtype=BF16, device=gpu)[1:].copy_(w)
    for q2 in (q.contiguous(), odd, bhsd, last):
        assert torch.equal(ops.norm_rope_kv_write(q2, k, v, pos, freq, w, w), want)
    for p2 in (pos.long(), pos.T.contiguous().T):
        assert torch.equal(ops.norm_rope_kv_write(q, k, v, p2, freq, w, w), want)
    for w1, w2 in ((w.float(), w.float()), (w.float(), w), (odd_w, odd_w)):
        assert torch.equal(ops.norm_rope_kv_write(q, k, v, pos, freq, w1, w2), want)
    one = q[:, :, :1].expand(-1, -1, Hq, -1)  # a broadcast head
    got = ops.norm_rope_kv_write(one, k, v, pos, freq, w, w)
    assert torch.equal(got, got[:, :, :1].expand_as(got))


def test_bad_numbers_stay_in_their_rows(gpu):
    B, S, H, D = 1, 6, 2, 128
    q, k, v = _inputs(gpu, B, S, H, H, D, BF16, 6, packed=False)
    pos = torch.arange(S, dtype=torch.int32, device=gpu)[None]
    freq, w = ops.rope_frequencies(D)[0].to(gpu), torch.ones(D, dtype=BF16, device=gpu)
    want = ops.norm_rope_kv_write(q, k, v, pos, freq, w, w)
    q[0, 2, 0, 5], q[0, 4, 1, 9] = float("nan"), float("inf")
    got = ops.norm_rope_kv_write(q, k, v, pos, freq, w, w)
    bad = torch.zeros(B, S, H, dtype=torch.bool, device=gpu)
    bad[0, 2, 0] = bad[0, 4, 1] = True
    assert torch.equal(got[~bad], want[~bad]) and got[0, 2, 0].isnan().all()
    q.zero_()
    assert (ops.norm_rope_kv_write(q, k, v, pos, freq, w, w) == 0).all()


@pytest.mark.parametrize("head_major", [False, True])
def test_pools_past_32_bits(gpu, head_major):
    """Rows at the end of pools of more than 2^31 elements, and at their start."""
    Hkv, D, page = 4, 128, 32
    pages = 2 ** 31 // (page * Hkv * D) + 7
    q, k, v = _inputs(gpu, 1, 6, 4, Hkv, D, BF16, 12)
    pos = torch.arange(6, dtype=torch.int32, device=gpu)[None]
    last = pages * page
    slots = torch.tensor([[last - 1, 0, last, last - 40, 2 ** 31 // (Hkv * D) + 1, 1]], device=gpu)
    shape = (pages, Hkv, page, D) if head_major else (pages, page, Hkv, D)
    pools = [torch.zeros(shape, dtype=BF16, device=gpu) for _ in range(2)]
    views = [p.transpose(1, 2) if head_major else p for p in pools]
    freq = ops.rope_frequencies(D)[0].to(gpu)
    _, k_got = ops.norm_rope_kv_write(q, k, v, pos, freq, k_cache=views[0], v_cache=views[1], slots=slots, kv_out=True)
    for c, rows in zip(views, (k_got, v)):
        for t, s in enumerate(slots[0].tolist()):
            if s < last:
                assert torch.equal(c[s // page, s % page], rows[0, t]), t
        assert int((c != 0).any(-1).any(-1).sum()) == 5


def test_empty(gpu):
    f = ops.rope_frequencies(64)[0].to(gpu)
    for B, S in ((0, 4), (3, 0)):
        q = torch.zeros(B, S, 2, 64, dtype=BF16, device=gpu)
        assert ops.norm_rope_kv_write(q, q, q, torch.zeros(B, S, dtype=torch.int32, device=gpu), f).shape == q.shape


def test_captured_and_on_another_stream(gpu):
    B, S, Hq, Hkv, D = 2, 8, 6, 2, 128
    q, k, v = (t.clone() for t in _inputs(gpu, B, S, Hq, Hkv, D, BF16, 8, packed=False))
    pos = torch.zeros(B, S, dtype=torch.int32, device=gpu)
    slots = torch.arange(B * S, device=gpu).view(B, S)
    freq, w = ops.rope_frequencies(D)[0].to(gpu), torch.ones(D, dtype=BF16, device=gpu)
    kc, vc = _pools(gpu, 2, 16, Hkv, D, BF16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.norm_rope_kv_write(q, k, v, pos, freq, w, w, 1e-6, kc, vc, slots)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = ops.norm_rope_kv_write(q, k, v, pos, freq, w, w, 1e-6, kc, vc, slots)
    for step in range(3):
        q.normal_()
        k.normal_()
        pos.fill_(step * 1000)
        slots.copy_(slots.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        kc2, vc2 = _pools(gpu, 2, 16, Hkv, D, BF16)
        want = ops.norm_rope_kv_write(q, k, v, pos, freq, w, w, 1e-6, kc2, vc2, slots)
        assert torch.equal(got, want) and torch.equal(kc[0], kc2[0]) and torch.equal(vc[0], vc2[0])


def test_refusals(gpu):
    q, k, v = _inputs(gpu, 2, 3, 4, 2, 64, BF16, 9)
    pos = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    f, w = ops.rope_frequencies(64)[0].to(gpu), torch.ones(64, dtype=BF16, device=gpu)
    kc, vc = _pools(gpu, 4, 16, 2, 64, BF16)
    slots = torch.zeros(2, 3, dtype=torch.int64, device=gpu)
    ok = dict(q=q, k=k, v=v, positions=pos, inv_freq=f)
    cache = dict(k_cache=kc, v_cache=vc, slots=slots)
    for kw in (dict(q=q[0]), dict(v=v[:, :2]), dict(k=k.half()), dict(q=q.double(), k=k.double(), v=v.double()),
               dict(positions=pos[:1]), dict(positions=pos.float()), dict(inv_freq=f.long()), dict(inv_freq=torch.ones(33, device=gpu)),
               dict(q_weight=w[:8]), dict(q_weight=w.half()), dict(k_cache=kc), dict(k_cache=kc, v_cache=vc), dict(slots=slots),
               dict(cache, slots=slots[:1]), dict(cache, slots=slots.float()), dict(cache, k_cache=kc[:, :, :1]),
               dict(cache, v_cache=vc[:2]), dict(cache, k_cache=kc.half()), dict(cache, k_cache=kc[:1].expand(4, -1, -1, -1)),
               dict(cache, k_cache=kc[:, :15], v_cache=vc[:, :15]),
               dict(cache, k_cache=torch.zeros(4 * 16 * 2 * 64 + 1, dtype=BF16, device=gpu)[1:].view(4, 16, 2, 64)),
               dict(q=q.cpu())):
        with pytest.raises(RuntimeError):
            ops.norm_rope_kv_write(**dict(ok, **kw))
    with pytest.raises(RuntimeError, match="backward"):
        ops.norm_rope_kv_write(**dict(ok, q=q.clone().requires_grad_()))
    with torch.no_grad():
        ops.norm_rope_kv_write(**dict(ok, q=q.clone().requires_grad_()))
    x = torch.zeros(1, 1, 1, 264, dtype=BF16, device=gpu)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.norm_rope_kv_write(x, x, x, pos[:1, :1], f)
