"""The operators of a step through the C++ host side (torch.ops.xllm_ops.*): the same bits as xllm_amd.ops, and refusals."""
import os
import subprocess
import sys

import pytest
import torch

from xllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def xops():
    from xllm_amd import torch_ops
    return torch_ops.load()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_step_tables(xops):
    kv, new, free, head = i32([5, 0, 33, 16]), i32([1, 20, 1, 0]), torch.arange(50, 90, dtype=torch.int32, device=DEV), i32([3])
    table = torch.randint(0, 50, (4, 6), device=DEV).to(torch.int32)
    want = ops.build_step_tables(kv, new, table, free, 16, 24, head)
    names = list(ops.StepTables.__dataclass_fields__)
    got = xops.build_step_tables(kv, new, table, free, 16, 24, head)
    for name, g in zip(names, got):
        assert torch.equal(g, getattr(want, name)), name
    outs = [torch.empty_like(g) for g in got]
    outs[0].copy_(table)
    xops.build_step_tables_out(kv, new, outs[0], free, 16, 24, head, *outs)   # the table in place
    for name, g in zip(names, outs):
        assert torch.equal(g, getattr(want, name)), name
    for bad in ((kv.long(), new, table, free, 16, 24), (kv, new[:3], table, free, 16, 24), (kv, new, table, free, 0, 24),
                (kv, new, table[:3], free, 16, 24), (kv, new, table, free.cpu(), 16, 24)):
        with pytest.raises((ValueError, TypeError)):
            xops.build_step_tables(*bad)


def test_rows_and_rotation(xops):
    inv, factor = ops.rope_frequencies(64, scaling=ops.RopeScaling("yarn", factor=4.0, original_max_position=64), device=DEV)
    pos = torch.randint(0, 300, (21,), device=DEV)
    rows = xops.build_cos_sin_cache(inv, None, 300, 0, factor, torch.float32)
    assert torch.equal(rows, ops.build_cos_sin_cache(inv, 300, attention_factor=factor))
    assert torch.equal(xops.build_cos_sin_cache(inv, pos, 0, 0, factor, torch.float32), rows[pos])
    q, k = torch.randn(21, 6, 96, device=DEV).to(BF16), torch.randn(21, 2, 64, device=DEV).to(BF16)
    for interleave in (False, True):
        for inverse in (False, True):
            want = ops.rotary_embedding(pos, q, k, rows, interleave=interleave, rotary_offset=32, key_rotary_offset=0,
                                        inverse=inverse, out_query=torch.empty_like(q), out_key=torch.empty_like(k))
            oq, ok, iq, ik = torch.empty_like(q), torch.empty_like(k), q.clone(), k.clone()
            xops.rotary_embedding(pos, q, k, rows, interleave, 32, 0, inverse, oq, ok)
            xops.rotary_embedding(pos, iq, ik, rows, interleave, 32, 0, inverse)
            for a, b in ((oq, want[0]), (ok, want[1]), (iq, want[0]), (ik, want[1])):
                assert torch.equal(a, b)
    alone = q.clone()
    xops.rotary_embedding(pos, alone, None, rows)
    assert torch.equal(alone, ops.rotary_embedding(pos, q.clone(), None, rows)[0])
    for bad in ((pos.int(), q, k, rows), (pos, q, k.float(), rows), (pos, q, k[:3], rows), (pos, q, k, rows.double()),
                (pos, q, q, rows), (pos, q.transpose(1, 2), None, rows)):
        with pytest.raises((ValueError, TypeError)):
            xops.rotary_embedding(*bad)
    with pytest.raises((ValueError, TypeError)):
        xops.build_cos_sin_cache(inv.float(), None, 10, 0, 1.0, torch.float32)
    with pytest.raises((ValueError, TypeError)):
        xops.build_cos_sin_cache(inv, None, 0, 0, 1.0, torch.float32)


def test_mla_prologue(xops):
    T, H = 9, 5
    q, kv, w = torch.randn(T, H, 192, device=DEV).to(BF16), torch.randn(T, 576, device=DEV).to(BF16), torch.ones(512, dtype=BF16, device=DEV)
    inv, _ = ops.rope_frequencies(64, device=DEV)
    rows, pos = ops.build_cos_sin_cache(inv, 50), torch.randint(0, 50, (T,), device=DEV)
    slots = torch.randperm(32, device=DEV)[:T].to(torch.int32)
    caches = [torch.zeros(2, 16, 1, 576, dtype=BF16, device=DEV) for _ in range(2)]
    oq = [torch.empty(T, H, 64, dtype=BF16, device=DEV) for _ in range(2)]
    okv = [torch.empty_like(kv) for _ in range(2)]
    ops.mla_norm_rope_and_cache(q[..., 128:], kv, w, 1e-6, rows, True, pos, k_cache=caches[0], slot_mapping=slots,
                                out_q_pe=oq[0], out_kv=okv[0])
    xops.mla_norm_rope_and_cache(q[..., 128:], kv, w, 1e-6, rows, True, pos, caches[1], slots, oq[1], okv[1])
    assert torch.equal(*caches) and torch.equal(*oq) and torch.equal(*okv)
    for change in (dict(slot_mapping=None), dict(k_cache=None), dict(kv=kv[:, :575]), dict(position_ids=pos.int()), dict(kv=kv.float())):
        args = dict(q_pe=q[..., 128:], kv=kv, kv_norm_weight=w, eps=1e-6, cos_sin_cache=rows, interleave=True, position_ids=pos,
                    k_cache=caches[0], slot_mapping=slots)
        args.update(change)
        with pytest.raises((ValueError, TypeError)):
            xops.mla_norm_rope_and_cache(**args)


def test_differential_decode(xops):
    B, H, pairs, D, bs, P = 3, 4, 2, 64, 16, 20
    q = torch.randn(B, 2 * H, D, device=DEV).to(BF16)
    k, v = torch.randn(P, bs, 2 * pairs, D, device=DEV).to(BF16), torch.randn(P, bs, pairs, 2 * D, device=DEV).to(BF16)
    table, lens = torch.randperm(P, device=DEV)[:18].view(3, 6).to(torch.int32), i32([90, 0, 17])
    lam, w = torch.rand(B, H, device=DEV), torch.ones(2 * D, dtype=BF16, device=DEV)
    want, got = torch.empty(B, H, 2 * D, dtype=BF16, device=DEV), torch.empty(B, H, 2 * D, dtype=BF16, device=DEV)
    for weight, window, lm in ((w, -1, lam), (None, 20, lam[0].contiguous()), (w, -1, lam[:1, :1])):
        ops.batch_decode_diff(q, k, v, want, table, lens, lm, scale=0.2, norm_weight=weight, eps=1e-6, out_scale=0.5, window_left=window)
        xops.batch_decode_diff(q, k, v, got, table, lens, lm, 0.2, weight, 1e-6, 0.5, window)
        assert torch.equal(got, want)
    for bad in ((q[:, :7], k, v, got, table, lens, lam, 0.2), (q, k, k, got, table, lens, lam, 0.2), (q, k, v, got, table, lens.long(), lam, 0.2),
                (q, k, v, got, table, lens, lam.double(), 0.2), (q, k, v, got.float(), table, lens, lam, 0.2), (q, k, v, got, table, lens, lam, -1.0)):
        with pytest.raises((ValueError, TypeError)):
            xops.batch_decode_diff(*bad)


_FIRST_CALLS = """
import threading, torch
from xllm_amd import ops
N, D, pairs = 8, 128, 2
dev = "cuda:0"
q = torch.randn(3, 8, D, device=dev).to(torch.float16)
k, v = torch.randn(40, 16, 2 * pairs, D, device=dev).half(), torch.randn(40, 16, pairs, 2 * D, device=dev).half()
table = torch.arange(39, device=dev).view(3, 13).to(torch.int32)
lens, lam = torch.tensor([200, 0, 33], dtype=torch.int32, device=dev), torch.rand(4, device=dev)
outs = [torch.zeros(3, 4, 2 * D, dtype=torch.float16, device=dev) for _ in range(N)]
ready, errors = threading.Barrier(N), []
torch.cuda.synchronize()

def first(out):
    try:
        ready.wait()
        with torch.cuda.stream(torch.cuda.Stream()):
            ops.batch_decode_diff(q, k, v, out, table, lens, lam)
    except Exception as e:
        errors.append(e)

threads = [threading.Thread(target=first, args=(o,)) for o in outs]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert not errors, errors
want = ops.batch_decode_diff(q, k, v, torch.empty_like(outs[0]), table, lens, lam)
assert all(torch.equal(o, want) for o in outs)
print("first calls agree")
"""


def test_first_calls_of_several_threads():
    """The first calls of a process come from eight threads at once: all of them find the kernel set up."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", _FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "first calls agree" in done.stdout, done.stdout + done.stderr


def test_results_count_as_written_in_place(xops):
    """A backward pass over values that a call has overwritten fails, as after torch's own in-place functions."""
    T, H, D = 3, 2, 64
    inv, _ = ops.rope_frequencies(D, device=DEV)
    rows, pos = ops.build_cos_sin_cache(inv, 8), torch.arange(T, device=DEV)
    for fn in (ops.rotary_embedding, xops.rotary_embedding):
        x = torch.randn(T, H, D, device=DEV, requires_grad=True)
        y = x.exp()   # (keeps its result for the backward pass)
        with torch.no_grad():
            fn(pos, y.detach(), None, rows)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()

    def versions(*tensors):
        return [t._version for t in tensors]

    kv, q = torch.zeros(T, 576, dtype=BF16, device=DEV), torch.zeros(T, H, D, dtype=BF16, device=DEV)
    cache, w = torch.zeros(1, 16, 1, 576, dtype=BF16, device=DEV), torch.ones(512, dtype=BF16, device=DEV)
    before = versions(q, kv, cache, w, rows, pos)
    ops.mla_norm_rope_and_cache(q, kv, w, 1e-6, rows, True, pos, k_cache=cache, slot_mapping=pos.int(), out_kv=kv)
    assert [a - b for a, b in zip(versions(q, kv, cache, w, rows, pos), before)] == [1, 1, 1, 0, 0, 0]
    out, key = torch.empty_like(q), torch.empty_like(q)
    before = versions(q, kv, rows, out, key)
    ops.rotary_embedding(pos, q, q.clone(), rows, out_query=out, out_key=key)
    ops.build_cos_sin_cache(inv, 8, out=rows)
    assert [a - b for a, b in zip(versions(q, kv, rows, out, key), before)] == [0, 0, 1, 1, 1]
    t = ops.build_step_tables(i32([1, 2]), i32([1, 1]), i32([[0, 1], [2, 3]]), i32([4, 5]), 16, 4)
    before = versions(t.block_table, t.slot_mapping, t.counters)
    ops.build_step_tables(i32([1, 2]), i32([1, 1]), i32([[0, 1], [2, 3]]), i32([4, 5]), 16, 4, out=t)
    assert all(a > b for a, b in zip(versions(t.block_table, t.slot_mapping, t.counters), before))
    lens, lam = i32([5]), torch.zeros(1, device=DEV)
    k, v, o = torch.zeros(1, 16, 2, D, dtype=BF16, device=DEV), torch.zeros(1, 16, 1, 2 * D, dtype=BF16, device=DEV), \
        torch.zeros(1, 1, 2 * D, dtype=BF16, device=DEV)
    before = versions(q, k, v, o)
    ops.batch_decode_diff(q[:1], k, v, o, i32([[0]]), lens, lam)
    assert [a - b for a, b in zip(versions(q, k, v, o), before)] == [0, 0, 0, 1]
    with torch.inference_mode():
        made = ops.build_cos_sin_cache(inv, 8)
        ops.rotary_embedding(pos, torch.zeros(T, H, D, device=DEV), None, made)
    ops.rotary_embedding(pos, torch.zeros(T, H, D, device=DEV), None, made)   # (a table made in inference mode, read outside)
