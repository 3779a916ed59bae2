"""The paged step's calls: the native host side against the Python statement of the same calls,
over the forms, and which forms it leaves to Python."""
import threading

import pytest
import torch

from fast_v2_amd import _ffi, ops
from test_host_calls_gpu import _both, _rnd, _same

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def _pool():
    return (torch.tensor([5, 0, 40], **I32), torch.zeros(3, 4, **I32), torch.arange(9, **I32), torch.tensor([9], **I32), 16)


@pytest.mark.parametrize("form", ["padded", "packed", "int64", "wide_table", "one", "strided_lens", "float", "shape",
                                  "neither", "page", "cpu", "itself"])
def test_pages(gpu, form):
    print(f"case pages {form}", flush=True)

    def make():
        new, pool = torch.tensor([3, 20, 1], **I32), list(_pool())
        kw = dict(rows=30) if form == "packed" else dict(width=32)
        if form == "int64":
            new = new.long()
        elif form == "wide_table":
            pool[1] = torch.zeros(3, 9, **I32)[:, :4]
        elif form == "one":
            new, pool[0], pool[1] = new[:1], pool[0][:1], pool[1][:1]
        elif form == "strided_lens":
            pool[0] = torch.zeros(6, **I32)[::2]
        elif form == "float":
            new = new.float()
        elif form == "shape":
            new = new[:2]
        elif form == "neither":
            kw = {}
        elif form == "page":
            pool[4] = 24
        elif form == "cpu":
            pool[2] = pool[2].cpu()
        elif form == "itself":  # as many again as there are
            new = pool[0]

        def fn():
            out = ops.assign_pages(new, *pool, **kw)
            keep = out.starts.long() if form == "int64" else pool[0] if form == "itself" else out.starts
            assert ops.release_pages(keep, *pool) is None
            return out
        return fn, pool
    left = {"int64": ("assign", "release"), "strided_lens": ("assign",), "float": ("assign",), "shape": ("assign",),
            "neither": ("assign",), "cpu": ("assign",), "itself": ("assign", "release")}
    _same(*_both(make, left.get(form, ())))


@pytest.mark.parametrize("form", ["plain", "no_norm", "one_norm", "fp32", "fp32_weights", "kv_out", "no_cache", "interleaved",
                                  "partial", "head_major", "int64", "unaligned", "mixed_weights", "f64_freq", "types", "slots32",
                                  "shape", "grad", "page", "empty"])
def test_norm_rope(gpu, form):
    print(f"case norm_rope {form}", flush=True)

    def make():
        dt = torch.float32 if form == "fp32" else torch.bfloat16
        x = _rnd(1, 2, 5, 8, 64, dtype=dt)
        a = dict(q=x[:, :, :4], k=x[:, :, 4:6], v=x[:, :, 6:], positions=torch.arange(10, **I32).view(2, 5),
                 inv_freq=torch.rand(32, device="cuda", generator=torch.Generator("cuda").manual_seed(1)), eps=1e-5,
                 q_weight=_rnd(2, 64, dtype=dt), k_weight=_rnd(3, 64, dtype=dt), slots=torch.arange(10, device="cuda").view(2, 5),
                 k_cache=torch.zeros(2, 16, 2, 64, device="cuda", dtype=dt), v_cache=torch.zeros(2, 16, 2, 64, device="cuda", dtype=dt))
        if form == "no_norm":
            a.update(q_weight=None, k_weight=None)
        elif form == "one_norm":
            a.update(q_weight=None)
        elif form == "fp32_weights":
            a.update(q_weight=a["q_weight"].float(), k_weight=a["k_weight"].float())
        elif form == "kv_out":
            a.update(kv_out=True)
        elif form == "no_cache":
            a.update(k_cache=None, v_cache=None, slots=None)
        elif form == "interleaved":
            a.update(interleaved=True, rope_scale=1.5)
        elif form == "partial":
            a.update(inv_freq=a["inv_freq"][:5])
        elif form == "head_major":
            a.update(k_cache=torch.zeros(2, 2, 16, 64, device="cuda", dtype=dt).transpose(1, 2))
        elif form == "int64":
            a.update(positions=a["positions"].long())
        elif form == "unaligned":
            a.update(q=_rnd(1, 2, 5, 4, 65)[..., 1:])
        elif form == "mixed_weights":
            a.update(q_weight=a["q_weight"].float())
        elif form == "f64_freq":
            a.update(inv_freq=a["inv_freq"].double())
        elif form == "types":
            a.update(k=a["k"].half())
        elif form == "slots32":
            a.update(slots=a["slots"].int())
        elif form == "shape":
            a.update(slots=a["slots"][:1])
        elif form == "grad":
            a.update(k_weight=torch.nn.Parameter(a["k_weight"]))
        elif form == "page":
            a.update(k_cache=a["k_cache"][:, :15], v_cache=a["v_cache"][:, :15])
        elif form == "empty":
            a.update({n: a[n][:0] for n in ("q", "k", "v", "positions", "slots")})
        return (lambda: ops.norm_rope_kv_write(**a)), [a["k_cache"], a["v_cache"]]
    left = form in ("int64", "unaligned", "mixed_weights", "f64_freq", "types", "slots32", "shape", "grad", "empty")
    _same(*_both(make, ("norm_rope",) if left else ()))


@pytest.mark.parametrize("form", ["2d", "3d", "1d", "4d", "many", "none", "shifted", "split", "strided", "int32", "outside",
                                  "types", "top", "tokens", "grad", "empty"])
def test_scores(gpu, form):
    print(f"case scores {form}", flush=True)

    def make():
        x, tok, k = _rnd(1, 6, 20, 700), torch.arange(120, device="cuda").view(6, 20), 3
        if form == "2d":
            x, tok = x[0], tok[0]
        elif form == "1d":
            x, tok = x[0, 0], tok[0, 0]
        elif form == "4d":
            x, tok = x.view(2, 3, 20, 700), tok.view(2, 3, 20)
        elif form == "many":
            tok, k = tok[..., None].expand(-1, -1, 4).contiguous(), 0
        elif form == "none":
            tok = None
        elif form == "shifted":
            x, tok = x[:, :-1], tok[:, 1:]
        elif form == "split":
            x, tok, k = _rnd(1, 2, 60000), tok[0, :2], 7
        elif form == "strided":
            x = _rnd(1, 6, 20, 1400)[..., ::2]
        elif form == "int32":
            tok = tok.int()
        elif form == "outside":
            tok = tok + 650
        elif form == "types":
            x = x.double()
        elif form == "top":
            k = 33
        elif form == "tokens":
            tok = tok[:, :3]
        elif form == "grad":
            x = x.requires_grad_()
        elif form == "empty":
            x, tok = x[:0], tok[:0]

        def fn():
            out = ops.token_logprobs(x, tok, k)
            return [torch.nan_to_num(t, nan=7.0) if t is not None and t.is_floating_point() else t for t in out]
        return fn, []
    left = form in ("4d", "shifted", "strided", "int32", "types", "top", "tokens", "grad", "empty")
    _same(*_both(make, ("logprobs",) if left else ()))


def test_a_non_current_device_is_made_current(gpu, monkeypatch):
    """The launch of a tensor's device that is not the current one happens inside a device guard."""
    seen = []

    class Guard:
        def __init__(self, dev):
            seen.append(dev)

        def __enter__(self):
            return self

        def __exit__(self, *a):
            pass
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(ops, "_HOST", type("Off", (), {"__getattr__": lambda self, name: lambda *a: None})())
    ops.token_logprobs(_rnd(1, 2, 50))
    pool = _pool()
    ops.release_pages(ops.assign_pages(torch.ones(3, **I32), *pool, width=1).starts, *pool)
    x = _rnd(1, 1, 1, 1, 8)
    ops.norm_rope_kv_write(x, x, x, torch.zeros(1, 1, **I32), torch.ones(4, device="cuda"))
    assert [d.index for d in seen] == [0] * 4


def test_threads(gpu):
    """Scores of two threads on one stream: each call's partial results are its own."""
    data = [(_rnd(i, 3, 40000 + 1000 * i), torch.arange(3, device="cuda")) for i in range(4)]
    want = [ops.token_logprobs(*a, 5) for a in data]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.Stream()] * 2):
        print(f"case threads, {len(set(streams))} streams", flush=True)
        bad, gate = [-1, -1], threading.Barrier(2)

        def run(i):
            with torch.cuda.stream(streams[i]):
                gate.wait()
                outs = [(j, ops.token_logprobs(*data[j], 5)) for _ in range(20) for j in range(4)]
                streams[i].synchronize()
                bad[i] = sum(not torch.equal(x, y) for j, o in outs for x, y in zip(o, want[j]))

        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert bad == [0, 0]


def test_inference_mode_and_wrappers(gpu):
    with torch.inference_mode():
        x = _rnd(1, 2, 700)
        out = ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64, device="cuda"), 2)
        assert out.entropy.is_inference()
    seen = []

    def fn(t):
        seen.append(ops._HOST.logprobs(t, None, 1))
        return t
    torch.vmap(fn)(_rnd(1, 3, 2, 50))
    assert seen == [None]


def test_wrapped_tensors_are_refused(gpu):
    """What carries more than its values: refused, not read without it."""
    import torch.autograd.forward_ad as fwd

    class Sub(torch.Tensor):
        pass
    x, i = _rnd(1, 1, 1, 2, 8), torch.zeros(1, 1, **I32)
    f = torch.ones(4, device="cuda")
    neg = torch._neg_view(x)
    assert neg.is_neg()
    for bad in (x.as_subclass(Sub), neg):
        with pytest.raises(RuntimeError, match="plain tensors"):
            ops.token_logprobs(bad)
        with pytest.raises(RuntimeError):
            ops.norm_rope_kv_write(bad, x, x, i, f)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="plain tensors"):
            ops.token_logprobs(fwd.make_dual(x.float(), x.float()))
    pool = list(_pool())
    pool[1] = pool[1].as_subclass(Sub)
    with pytest.raises(RuntimeError, match="plain tensors"):
        ops.assign_pages(torch.ones(3, **I32), *pool, width=1)
