"""The operators around the paged cache without a GPU: the oracle's closed forms, the
frequencies, and what the calls refuse (through the C ABI too, before any launch)."""
import ctypes
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from fast_v2_amd import _ffi, ops
from oracle import paged_step as ps

ROOT = Path(__file__).resolve().parents[1]


# ---- the oracle ------------------------------------------------------------------------

def test_oracle_pages_by_hand():
    table = np.zeros((3, 4), np.int64)
    table[0, 0] = 9
    lens, free = [3, 0, 8], [1, 2, 3, 4, 5]
    table[2, :2] = [7, 8]
    out = ps.assign_pages_np([2, 5, 1], lens, table, free, 4, rows=9)
    assert lens == [5, 5, 9] and free == [1]
    assert table.tolist() == [[9, 5, 0, 0], [4, 3, 0, 0], [7, 8, 2, 0]]
    assert out["slots"].tolist() == [39, 20, 16, 17, 18, 19, 12, 8, -1]
    assert out["positions"].tolist() == [3, 4, 0, 1, 2, 3, 4, 8, 0]
    assert out["sequences"].tolist() == [0, 0, 1, 1, 1, 1, 1, 2, -1] and out["row_starts"] == [0, 2, 7, 8]
    ps.release_pages_np(out["starts"], lens, table, free, 4)
    assert lens == [3, 0, 8] and free == [1, 2, 3, 4, 5]


def test_oracle_pages_run_out_in_order():
    table, lens, free = np.zeros((4, 4), np.int64), [0, 0, 3, 0], [6]
    out = ps.assign_pages_np([4, 5, 1, 1], lens, table, free, 4, width=8)
    # the first takes the page, the second finds too few, the third has room, the fourth comes too late
    assert out["granted"] == [4, 0, 1, 0] and lens == [4, 0, 4, 0] and free == []
    assert out["slots"].reshape(4, 8)[2].tolist() == [3] + [-1] * 7


def test_oracle_rotation_closed_forms():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((1, 3, 2, 8))
    f = np.array([1.0, 0.5, 0.25])
    assert np.array_equal(ps.norm_rope_np(x, np.zeros((1, 3)), f), x)
    y = ps.norm_rope_np(x, np.full((1, 3), 2.0), f)
    for i, a in enumerate(2 * f):
        want = x[..., i] * math.cos(a) - x[..., i + 3] * math.sin(a)
        np.testing.assert_allclose(y[..., i], want, atol=1e-14)
    assert np.array_equal(y[..., 6:], x[..., 6:])
    z = ps.norm_rope_np(x, np.full((1, 3), 2.0), f, interleaved=True)
    np.testing.assert_allclose(z[..., 3], x[..., 3] * math.cos(1) + x[..., 2] * math.sin(1), atol=1e-14)
    n = ps.norm_rope_np(x, np.zeros((1, 3)), f, weight=np.ones(8), eps=0.0)
    np.testing.assert_allclose((n * n).mean(-1), 1.0, atol=1e-14)


def test_oracle_scores_closed_forms():
    x = np.zeros((3, 10))
    x[1, 4] = -np.inf
    x[2] = np.arange(10)
    lp, ent, top, ids = ps.token_logprobs_np(x, np.array([[0, 11], [4, 5], [9, 0]]), 3)
    np.testing.assert_allclose(lp[0, 0], -math.log(10))
    assert np.isnan(lp[0, 1]) and lp[1, 0] == -np.inf
    np.testing.assert_allclose(ent[:2], [math.log(10), math.log(9)])
    assert ids.tolist() == [[0, 1, 2], [0, 1, 2], [9, 8, 7]]
    np.testing.assert_allclose(top[2, 1] - top[2, 0], -1.0)
    assert np.isnan(ps.token_logprobs_np(np.full((1, 4), -np.inf), None, 1)[1]).all()


# ---- frequencies -----------------------------------------------------------------------

def test_frequencies():
    f, scale = ops.rope_frequencies(8, base=10000.0)
    assert scale == 1.0 and f.dtype == torch.float32
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001]), rtol=2 ** -24 * 4, atol=0)
    torch.testing.assert_close(ops.rope_frequencies(8, 10000.0, "linear", 4.0)[0], f / 4)
    n = ops.rope_frequencies(8, 10000.0, "ntk", 4.0)[0]
    torch.testing.assert_close(n[[0, -1]], torch.stack([f[0], f[-1] / 4]))  # fastest kept, slowest by the factor
    y, scale = ops.rope_frequencies(64, 10000.0, "yarn", 8.0, original_len=4096)
    plain = ops.rope_frequencies(64, 10000.0)[0]
    turns = 4096 * plain.double() / (2 * math.pi)
    assert scale == pytest.approx(0.1 * math.log(8) + 1)
    assert torch.equal(y[turns >= 32.1], plain[turns >= 32.1])
    torch.testing.assert_close(y[turns <= 0.99], plain[turns <= 0.99] / 8)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((y < plain) & (y > plain / 8))[between].all()
    assert ops.rope_frequencies(0)[0].numel() == 0
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(RuntimeError):
            ops.rope_frequencies(**bad)


# ---- refusals --------------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.assign_pages(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], 16, width=1)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.release_pages(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], 16)
    x = torch.zeros(1, 1, 1, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.norm_rope_kv_write(x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.ones(4))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.token_logprobs(torch.zeros(2, 8))


def test_sizes_past_32_bits_are_refused():
    """The descriptors' fields would wrap them: 2^32 + 16 is no page size of 16."""
    i, table, far = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32), 2 ** 32 + 16
    for kw in (dict(page_size=far, width=1), dict(page_size=16, width=far), dict(page_size=16, rows=far),
               dict(page_size=16, width=2 ** 30)):
        with pytest.raises(RuntimeError, match="too large"):
            ops.assign_pages(i, i, table, i, i[:1], **kw)
    for args in ((table, i, far), (i[:1, None].expand(2, far), i, 16), (table, i[:1].expand(far), 16)):
        with pytest.raises(RuntimeError, match="too large"):
            ops.release_pages(i, i, args[0], args[1], i[:1], args[2])
    f, one = torch.ones(4), torch.zeros(1, 1, 1, 8)
    for shape in ((far, 1, 1, 8), (1, far, 1, 8)):
        x = one.expand(shape)
        with pytest.raises(RuntimeError, match="too large"):
            ops.norm_rope_kv_write(x, x, x, i[:1].expand(shape[:2]), f)
    with pytest.raises(RuntimeError, match="too large"):
        ops.norm_rope_kv_write(one.expand(1, 1, far, 8), one, one, i[:1, None], f)
    pool = one.expand(1, far, 1, 8)
    with pytest.raises(RuntimeError, match="too large"):
        ops.norm_rope_kv_write(one, one, one, i[:1, None], f, k_cache=pool, v_cache=pool, slots=i[:1, None])
    for shape in ((far,), (2, far), (far, 2), (far, 2, 2)):
        with pytest.raises(RuntimeError, match="too large"):
            ops.token_logprobs(torch.zeros(1).expand(shape))
    with pytest.raises(RuntimeError, match="too large"):
        ops.token_logprobs(torch.zeros(2, 8), i[:1].expand(2, far))


@pytest.fixture(scope="module")
def lib():
    if not _ffi.LIB_PATH.exists():
        pytest.fail(f"{_ffi.LIB_PATH} is not built (run __graft_entry__.build())")
    return _ffi.lib()


def test_c_abi_refuses_bad_pools(lib):
    def pool(**kw):
        p = _ffi.PagePool(16, 4, 16, 16, 16, 2, 4, 8, 16)
        for name, v in kw.items():
            setattr(p, name, v)
        return p

    def assign(p, width=1, rows=0, seq=None):
        return lib.fdllm_assign_pages(ctypes.byref(p) if p else None, 16, width, rows, 16, 16, seq, seq, 16, 16, 16, 16, None)
    bad = _ffi.FDLLM_ERR_INVALID_ARGUMENT
    for kw in (dict(requests=-1), dict(requests=8193), dict(page_size=0), dict(page_size=24), dict(max_pages=-1),
               dict(num_free=-1), dict(table_stride=3), dict(lens=None), dict(free_count=None), dict(page_table=None),
               dict(free_pages=None)):
        assert assign(pool(**kw)) == bad, kw
        assert lib.fdllm_release_pages(ctypes.byref(pool(**kw)), 16, None) == bad, kw
    assert assign(None) == bad and lib.fdllm_release_pages(None, 16, None) == bad
    assert assign(pool(), 1, 1) == bad and assign(pool(), -1) == bad and assign(pool(), 0, -1) == bad
    assert assign(pool(), 0, 0, 16) == bad and assign(pool(), 2 ** 30) == bad and assign(pool(), 0, 2 ** 31 - 1, 16) == bad
    assert assign(pool(), 0, 4) == bad  # the packed form without its two outputs
    assert assign(pool(requests=0), 0, 4, 16) == bad
    assert assign(pool(requests=0)) == 0 and lib.fdllm_release_pages(ctypes.byref(pool(requests=0)), None, None) == 0
    assert lib.fdllm_release_pages(ctypes.byref(pool()), None, None) == bad


def test_c_abi_refuses_bad_rows(lib):
    def call(**kw):
        d = _ffi.NormRopeKVDesc()
        d.q = d.k = d.v = d.q_out = d.positions = d.inv_freq = d.k_cache = d.v_cache = d.slots = 64
        d.batch = d.seq_len = d.num_kv_heads = 1
        d.num_q_heads, d.head_dim, d.rotary_dim, d.dtype, d.weight_dtype = 2, 64, 64, _ffi.DTYPE_BF16, _ffi.DTYPE_BF16
        d.page_size, d.num_pages = 16, 4
        for name, v in kw.items():
            setattr(d, name, v)
        return lib.fdllm_norm_rope_kv_write(ctypes.byref(d), None)
    bad = _ffi.FDLLM_ERR_INVALID_ARGUMENT
    for kw in (dict(dtype=9), dict(weight_dtype=_ffi.DTYPE_F16), dict(head_dim=60), dict(head_dim=264), dict(rotary_dim=66),
               dict(rotary_dim=7), dict(rotary_dim=-2), dict(num_q_heads=0), dict(num_kv_heads=0), dict(batch=-1),
               dict(q=None), dict(v=None), dict(positions=None), dict(inv_freq=None), dict(slots=None), dict(k_cache=None),
               dict(page_size=24), dict(page_size=0), dict(num_pages=-1), dict(q=68), dict(k_cache=72), dict(q_weight=8),
               dict(q_stride_h=4), dict(v_stride_page=7), dict(batch=1 << 20, seq_len=1 << 20)):
        assert call(**kw) == bad, kw
    assert call(batch=0) == 0 and call(seq_len=0) == 0
    assert lib.fdllm_norm_rope_kv_write(None, None) == bad


def test_c_abi_refuses_bad_scores(lib):
    size = ctypes.c_size_t(1)

    def need(v, rows, dt):
        return lib.fdllm_token_logprobs_workspace_size(v, rows, dt, ctypes.byref(size))

    def call(batch=1, rows=1, vocab=100, given=0, top=0, logits=64, tokens=None, top_out=None, dt=_ffi.DTYPE_BF16, ws=None):
        return lib.fdllm_token_logprobs(logits, 0, 0, batch, rows, vocab, tokens, given, top, tokens, 64, top_out, top_out,
                                        dt, ws, 0, None)
    bad = _ffi.FDLLM_ERR_INVALID_ARGUMENT
    assert need(0, 1, 1) == bad and need(1 << 22, 1, 1) == bad and need(8, -1, 1) == bad and need(8, 1, 7) == bad
    assert lib.fdllm_token_logprobs_workspace_size(8, 1, 1, None) == bad
    assert need(152064, 1, 0) == 0 and size.value > 0
    assert need(152064, 100000, 1) == 0 and size.value == 0
    assert need(152064, 0, 1) == 0 and size.value == 0
    for kw in (dict(batch=-1), dict(vocab=0), dict(dt=5), dict(top=33, top_out=64), dict(top=4), dict(given=1), dict(given=-1),
               dict(logits=None), dict(vocab=3, top=4, top_out=64), dict(batch=1 << 16, rows=1 << 16)):
        assert call(**kw) == bad, kw
    assert call(vocab=152064) == _ffi.FDLLM_ERR_WORKSPACE
    assert call(batch=0) == 0


def test_c_abi_refuses_more_than_a_launch_holds(lib):
    """A launch has fewer than 2^32 threads: 64 a token, 256 a row."""
    bad, size = _ffi.FDLLM_ERR_INVALID_ARGUMENT, ctypes.c_size_t(0)
    d = _ffi.NormRopeKVDesc()
    d.q = d.k = d.v = d.q_out = d.positions = d.inv_freq = 64
    d.num_q_heads, d.num_kv_heads, d.head_dim, d.rotary_dim = 1, 1, 8, 8
    d.dtype = d.weight_dtype = _ffi.DTYPE_BF16
    for d.batch, d.seq_len in ((1 << 13, 1 << 13), (1, 1 << 26)):
        assert lib.fdllm_norm_rope_kv_write(ctypes.byref(d), None) == bad
        assert b"tokens" in lib.fdllm_last_error()
    assert lib.fdllm_token_logprobs_workspace_size(8, 1 << 24, _ffi.DTYPE_BF16, ctypes.byref(size)) == bad
    assert lib.fdllm_token_logprobs_workspace_size(8, (1 << 24) - 1, _ffi.DTYPE_BF16, ctypes.byref(size)) == 0
    assert lib.fdllm_token_logprobs(64, 8, 8, 1 << 12, 1 << 12, 8, None, 0, 0, None, 64, None, None, _ffi.DTYPE_BF16, None,
                                    0, None) == bad


@pytest.mark.parametrize("struct,mirror", [("fdllm_page_pool", _ffi.PagePool),
                                           ("fdllm_norm_rope_kv_desc", _ffi.NormRopeKVDesc)])
def test_descriptors_match_the_c_compiler(tmp_path, struct, mirror):
    fields = [f[0] for f in mirror._fields_]
    prog = tmp_path / "layout.c"
    prog.write_text("\n".join(
        ['#include <stdio.h>', '#include <stddef.h>', f'#include "{ROOT / "include" / "fdllm_hip.h"}"', 'int main(void) {',
         f'  printf("size %zu\\n", sizeof({struct}));']
        + [f'  printf("{n} %zu\\n", offsetof({struct}, {n}));' for n in fields] + ['  return 0;', '}']) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(prog)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(mirror)
    for n in fields:
        assert int(got[n]) == getattr(mirror, n).offset, n
