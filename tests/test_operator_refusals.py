"""What the step-table, rotary, MLA-prologue and differential entry points refuse before anything is launched: no GPU."""
import ctypes

import pytest
import torch

from xllm_amd import capi, ops

FAKE = 1 << 20   # an aligned non-null address: the calls below return before anything is launched
APART = [1 << (24 + i) for i in range(16)]   # aligned addresses whose tensors do not meet
BF16, FP16, FP32, FP8 = capi.BF16, capi.FP16, capi.FP32, capi.FP8_E4M3
EINVAL, EDTYPE, ESHAPE, EWORKSPACE, EALIGN = -1, -2, -3, -4, -5


def strides(a, b):
    return (ctypes.c_int64 * 2)(a, b)


def call(fn, base, **change):
    args = dict(base)
    assert set(change) <= set(args)
    args.update(change)
    return fn(*args.values())


def test_step_tables():
    fn = capi.lib().xllm_mi355_build_step_tables
    base = dict(kv=FAKE, new=FAKE, tin=FAKE, in_stride=8, tout=FAKE, out_stride=8, width=8, free=FAKE, n_free=9, head=None,
                seq=FAKE, cu=FAKE, pos=FAKE, slots=FAKE, indptr=FAKE, counters=FAKE, batch=4, bs=16, budget=8, stream=None)
    assert call(fn, base, batch=0) == 0
    for name in ("kv", "new", "tin", "tout", "free", "seq", "cu", "pos", "slots", "indptr", "counters"):
        assert call(fn, base, **{name: None}) == EINVAL, name
    for change in (dict(batch=-1), dict(bs=0), dict(width=0), dict(n_free=-1), dict(budget=-1), dict(in_stride=7),
                   dict(out_stride=7), dict(out_stride=9)):   # (in place with another stride)
        assert call(fn, base, **change) == EINVAL, change
    for change in (dict(budget=1 << 30), dict(n_free=1 << 30), dict(bs=1 << 30), dict(batch=(1 << 20) + 1)):
        assert call(fn, base, **change) == ESHAPE, change


def test_an_empty_batch_leaves_the_results_alone():
    """No requests: the C entry writes nothing, as its header says (host memory here; a write would be seen)."""
    fn = capi.lib().xllm_mi355_build_step_tables
    outs = [torch.full((n,), 77, dtype=dt) for n, dt in ((8, torch.int32), (1, torch.int32), (1, torch.int32), (8, torch.int64),
                                                         (8, torch.int32), (1, torch.int32), (3, torch.int32))]
    table, seq, cu, pos, slots, indptr, counters = (o.data_ptr() for o in outs)
    lens, free, head = torch.zeros(1, dtype=torch.int32), torch.arange(9, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    assert fn(lens.data_ptr(), lens.data_ptr(), table, 8, table, 8, 8, free.data_ptr(), 9, head.data_ptr(), seq, cu, pos, slots,
              indptr, counters, 0, 16, 8, None) == 0
    assert all((o == 77).all() for o in outs)


def test_cos_sin_rows():
    fn = capi.lib().xllm_mi355_rope_cos_sin
    base = dict(inv=FAKE, pos=None, first=0, rows=4, half=32, factor=1.0, out=FAKE, dtype=FP32, stream=None)
    assert call(fn, base, rows=0) == 0
    for change in (dict(inv=None), dict(out=None), dict(rows=-1), dict(half=0)):
        assert call(fn, base, **change) == EINVAL, change
    assert call(fn, base, half=4097) == ESHAPE
    assert call(fn, base, dtype=FP8) == EDTYPE


def test_rotation():
    fn = capi.lib().xllm_mi355_rotary_embedding
    st = strides(512, 128)
    base = dict(pos=FAKE, table=FAKE, rows=10, q=FAKE, qo=FAKE, k=FAKE, ko=FAKE, T=4, hq=4, hk=4, dq=128, dk=128, oq=0, ok=0,
                R=64, sq=st, sqo=st, sk=st, sko=st, interleave=0, inverse=0, dtype=BF16, ctype=FP32, stream=None)
    assert call(fn, base, T=0) == 0
    for change in (dict(pos=None), dict(table=None), dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(sq=None),
                   dict(sqo=None), dict(sk=None), dict(sko=None), dict(T=-1), dict(rows=0), dict(hq=0), dict(hk=-1),
                   dict(sq=strides(-512, 128)), dict(sqo=strides(640, 128))):   # (in place with other strides)
        assert call(fn, base, **change) == EINVAL, change
    for change in (dict(R=0), dict(R=63), dict(oq=65), dict(ok=-1), dict(ok=70), dict(R=256), dict(hq=65536)):
        assert call(fn, base, **change) == ESHAPE, change
    for change in (dict(dtype=FP8), dict(ctype=FP8)):
        assert call(fn, base, **change) == EDTYPE, change


def test_mla_prologue():
    fn = capi.lib().xllm_mi355_mla_norm_rope_and_cache
    base = dict(q=FAKE, qo=FAKE, kv=FAKE, kvo=None, w=FAKE, eps=1e-6, table=FAKE, rows=10, pos=FAKE, cache=FAKE, slots=FAKE,
                T=4, H=8, dl=512, dr=64, qt=1536, qh=192, qot=512, qoh=64, kvs=576, kvos=0, bs=16, P=4, interleave=1,
                dtype=BF16, ctype=FP32, stream=None)
    assert call(fn, base, T=0) == 0
    for change in (dict(q=None), dict(qo=None), dict(kv=None), dict(w=None), dict(table=None), dict(pos=None), dict(cache=None),
                   dict(slots=None), dict(T=-1), dict(H=0), dict(rows=0), dict(bs=0), dict(P=0), dict(kvs=575),
                   dict(kvo=FAKE, kvos=512), dict(eps=-1.0), dict(qt=-8)):
        assert call(fn, base, **change) == EINVAL, change
    for change in (dict(dl=256), dict(dr=32), dict(P=1 << 28)):
        assert call(fn, base, **change) == ESHAPE, change
    assert call(fn, base, dtype=FP32) == EDTYPE and call(fn, base, ctype=FP8) == EDTYPE
    for change in (dict(q=FAKE + 2), dict(qo=FAKE + 8), dict(kv=FAKE + 4), dict(w=FAKE + 2), dict(table=FAKE + 4),
                   dict(cache=FAKE + 8), dict(qt=1540), dict(qh=66), dict(kvs=577), dict(kvo=FAKE, kvos=580)):
        assert call(fn, base, **change) == EALIGN, change


def test_launches_beyond_32_bits_of_threads():
    lib = capi.lib()
    far = [1 << 44, 1 << 45, 1 << 46, 1 << 47, 1 << 48]   # (apart from each other by more than the largest operand)
    assert lib.xllm_mi355_rope_cos_sin(far[0], None, 0, 1 << 33, 1, 1.0, far[1], FP32, None) == ESHAPE
    assert lib.xllm_mi355_rope_cos_sin(far[0], None, 0, 1 << 28, 64, 1.0, far[1], FP32, None) == ESHAPE
    st = strides(64 * 64 + 1, 64)   # (not aligned: a lane per pair)
    assert lib.xllm_mi355_rotary_embedding(far[0], far[1], 10, far[2], far[2], None, None, 1 << 22, 64, 0, 64, 0, 0, 0, 64, st, st,
                                           None, None, 0, 0, BF16, FP32, None) == ESHAPE
    assert lib.xllm_mi355_mla_norm_rope_and_cache(far[0], far[0], far[1], far[1], far[2], 1e-6, far[3], 10, far[4], None, None,
                                                  1 << 23, 128, 512, 64, 8192, 64, 8192, 64, 576, 576, 16, 4, 1, BF16, FP32,
                                                  None) == ESHAPE


def test_differential_decode():
    lib = capi.lib()
    size = lib.xllm_mi355_paged_decode_diff_workspace_bytes
    assert size(16, 4, 64) > 0 and 0 < size(16, 4, 128) < size(64, 4, 128)
    assert size(0, 1, 128) == 0 and size(5, 2, 128) == 0 and size(4, 2, 96) == 0
    fn = lib.xllm_mi355_paged_decode_diff
    base = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, table=FAKE, stride=8, width=8, lens=FAKE, lam=FAKE, lb=0, lh=1, w=None,
                eps=1e-5, out_scale=1.0, batch=4, H=16, pairs=4, D=128, bs=16, P=100, qs=4096, os=4096, window=-1, scale=0.1,
                ws=FAKE, ws_bytes=size(16, 4, 128), dtype=BF16, stream=None)
    assert call(fn, base, batch=0) == 0
    for name in ("q", "k", "v", "out", "table", "lens", "lam"):
        assert call(fn, base, **{name: None}) == EINVAL, name
    for change in (dict(batch=-1), dict(H=0), dict(pairs=3), dict(bs=0), dict(P=0), dict(width=0), dict(stride=7),
                   dict(scale=0.0), dict(scale=float("nan")), dict(eps=-1.0), dict(lb=-1), dict(lh=-1), dict(qs=4095), dict(os=2048)):
        assert call(fn, base, **change) == EINVAL, change
    for change in (dict(D=96), dict(D=256), dict(P=1 << 28)):
        assert call(fn, base, **change) == ESHAPE, change
    # tables that could hold more stages of one sequence than 32 bits count; a window bounds them
    vast = dict(H=256, pairs=256, qs=65536, os=65536, bs=1 << 20, P=1, width=2048, stride=2048)
    assert call(fn, base, **vast) == ESHAPE
    assert call(fn, base, **vast, window=100, ws=None) == EWORKSPACE
    for dtype in (FP32, FP8):
        assert call(fn, base, dtype=dtype) == EDTYPE
    for change in (dict(q=FAKE + 8), dict(k=FAKE + 2), dict(v=FAKE + 8), dict(out=FAKE + 4), dict(w=FAKE + 4), dict(qs=4100),
                   dict(os=4097)):
        assert call(fn, base, **change) == EALIGN, change
    for change in (dict(ws=None), dict(ws=FAKE + 64), dict(ws_bytes=size(16, 4, 128) - 1)):
        assert call(fn, base, **change) == EWORKSPACE, change


def test_outputs_that_meet_inputs_or_each_other():
    """Addresses far apart, then one output moved onto each of the other operands in turn."""
    lib = capi.lib()

    def spread(base, names):
        at = dict(zip(names, APART))
        return dict(base, **at), at

    st = strides(512, 128)
    tables, at = spread(dict(kv=0, new=0, tin=0, in_stride=8, tout=0, out_stride=8, width=8, free=0, n_free=9, head=0, seq=0,
                             cu=0, pos=0, slots=0, indptr=0, counters=0, batch=4, bs=16, budget=8, stream=None),
                        ("kv", "new", "tin", "tout", "free", "head", "seq", "cu", "pos", "slots", "indptr", "counters"))
    for out in ("tout", "seq", "cu", "pos", "slots", "indptr", "counters"):
        for other in at:
            if other != out and (out, other) != ("tout", "tin"):
                got = call(lib.xllm_mi355_build_step_tables, tables, **{out: at[other]})
                assert got == EINVAL, (out, other)
    assert call(lib.xllm_mi355_build_step_tables, tables, tout=at["tin"] + 4) == EINVAL
    rot, at = spread(dict(pos=0, table=0, rows=10, q=0, qo=0, k=0, ko=0, T=4, hq=4, hk=4, dq=128, dk=128, oq=0, ok=0, R=64,
                          sq=st, sqo=st, sk=st, sko=st, interleave=0, inverse=0, dtype=BF16, ctype=FP32, stream=None),
                     ("pos", "table", "q", "qo", "k", "ko"))
    for out, others in (("qo", ("pos", "table", "k", "ko")), ("ko", ("pos", "table", "q", "qo"))):
        for other in others:
            assert call(lib.xllm_mi355_rotary_embedding, rot, **{out: at[other]}) == EINVAL, (out, other)
    assert call(lib.xllm_mi355_rotary_embedding, rot, qo=at["q"] + 16) == EINVAL
    assert call(lib.xllm_mi355_rotary_embedding, rot, qo=at["q"], sqo=strides(512, 64)) == EINVAL   # heads meet
    assert call(lib.xllm_mi355_rotary_embedding, rot, sqo=strides(256, 128)) == EINVAL              # tokens meet
    # two operands of one buffer whose rows meet: four heads each of [T, 7, 128], in place; results that meet by one word
    st = strides(7 * 128, 128)
    one = dict(rot, qo=at["q"], k=at["q"] + 3 * 256, ko=at["q"] + 3 * 256, sq=st, sqo=st, sk=st, sko=st)
    assert call(lib.xllm_mi355_rotary_embedding, one) == EINVAL
    assert call(lib.xllm_mi355_rotary_embedding, dict(one, ko=at["ko"])) == EINVAL   # (k is read where q is written)
    st = strides(8 * 128 - 8, 128)
    two = dict(rot, ko=at["qo"] + 4 * 256, sqo=st, sko=st)
    assert call(lib.xllm_mi355_rotary_embedding, two) == EINVAL
    for where in ("pos", "table"):
        assert call(lib.xllm_mi355_rotary_embedding, rot, qo=at[where], q=at[where]) == EINVAL, where
    mla, at = spread(dict(q=0, qo=0, kv=0, kvo=0, w=0, eps=1e-6, table=0, rows=10, pos=0, cache=0, slots=0, T=4, H=8, dl=512,
                          dr=64, qt=1536, qh=192, qot=512, qoh=64, kvs=576, kvos=576, bs=16, P=4, interleave=1, dtype=BF16,
                          ctype=FP32, stream=None),
                     ("q", "qo", "kv", "kvo", "w", "table", "pos", "cache", "slots"))
    for out in ("qo", "kvo", "cache"):
        for other in at:
            if other != out and (out, other) != ("kvo", "kv"):
                got = call(lib.xllm_mi355_mla_norm_rope_and_cache, mla, **{out: at[other]})
                assert got == EINVAL, (out, other)
    assert call(lib.xllm_mi355_mla_norm_rope_and_cache, mla, kvo=at["kv"] + 16) == EINVAL
    # latent rows and rope parts of one buffer of 1936 values a token: the last head meets the next token's latent
    fused = dict(mla, q=at["kv"] + 1152 + 16, qo=at["kv"] + 1152 + 16, qt=1936, qot=1936, qh=192, qoh=192, kvs=1936, kvos=1936)
    assert call(lib.xllm_mi355_mla_norm_rope_and_cache, fused, kvo=at["kv"]) == EINVAL
    rows, at = spread(dict(inv=0, pos=0, first=0, rows=4, half=32, factor=1.0, out=0, dtype=FP32, stream=None), ("inv", "pos", "out"))
    for other in ("inv", "pos"):
        assert call(lib.xllm_mi355_rope_cos_sin, rows, out=at[other]) == EINVAL
    need = lib.xllm_mi355_paged_decode_diff_workspace_bytes(4, 2, 64)
    diff, at = spread(dict(q=0, k=0, v=0, out=0, table=0, stride=8, width=8, lens=0, lam=0, lb=0, lh=1, w=0, eps=1e-5,
                           out_scale=1.0, batch=2, H=4, pairs=2, D=64, bs=16, P=4, qs=512, os=512, window=-1, scale=0.1,
                           ws=0, ws_bytes=need, dtype=BF16, stream=None),
                      ("q", "k", "v", "out", "table", "lens", "lam", "w", "ws"))
    diff["ws"] = at["ws"] = 1 << 45
    for out in ("out", "ws"):
        for other in at:
            if other != out:
                assert call(lib.xllm_mi355_paged_decode_diff, diff, **{out: at[other]}) == EINVAL, (out, other)


def test_cpu_tensors_are_refused():
    i32 = torch.int32
    one = torch.zeros(1, dtype=i32)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    rows = torch.zeros(4, 64)
    pos = torch.zeros(1, dtype=torch.int64)
    calls = [lambda: ops.build_step_tables(one, one, torch.zeros(1, 2, dtype=i32), one, 16, 1),
             lambda: ops.build_cos_sin_cache(torch.ones(4, dtype=torch.float64), 3),
             lambda: ops.rotary_embedding(pos, q, None, rows),
             lambda: ops.mla_norm_rope_and_cache(q, torch.zeros(1, 576), torch.ones(512), 1e-6, rows, True, pos),
             lambda: ops.batch_decode_diff(q, q, q, q, one, one, rows)]
    for c in calls:
        with pytest.raises(ValueError, match="GPU only"):
            c()


def test_frequencies_need_no_gpu():
    inv, factor = ops.rope_frequencies(64, scaling=ops.RopeScaling("linear", factor=2.0), device="cpu")
    assert inv.dtype == torch.float64 and inv[0] == 0.5 and factor == 1.0


def test_operands_that_require_grad_are_refused_while_a_graph_is_recorded():
    """No operator records a graph, so a gradient would be lost without a word.  (Under no_grad the call goes on, to the
    refusal of host tensors.)"""
    def grad(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, requires_grad=True)

    def plain(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype)

    pos, rows, slots = torch.zeros(1, dtype=torch.int64), torch.zeros(4, 64), torch.zeros(1, dtype=torch.int32)
    rot = dict(position_ids=pos, query=plain(1, 2, 64), key=plain(1, 2, 64), cos_sin_cache=rows, out_query=plain(1, 2, 64),
               out_key=plain(1, 2, 64))
    mla = dict(q_pe=plain(1, 2, 64), kv=plain(1, 576), kv_norm_weight=plain(512), eps=1e-6, cos_sin_cache=rows, interleave=True,
               position_ids=pos, k_cache=plain(1, 16, 1, 576), slot_mapping=slots, out_q_pe=plain(1, 2, 64), out_kv=plain(1, 576))
    diff = dict(query=plain(1, 2, 64), k_cache=plain(1, 16, 2, 64), v_cache=plain(1, 16, 1, 128), output=plain(1, 1, 128),
                block_table=slots.view(1, 1), seq_lens=slots, lambda_=torch.zeros(1), norm_weight=plain(128))
    angles = dict(inv_freq=torch.ones(4, dtype=torch.float64), num_positions=3, out=torch.zeros(3, 8))
    for fn, base in ((ops.rotary_embedding, rot), (ops.mla_norm_rope_and_cache, mla), (ops.batch_decode_diff, diff),
                     (ops.build_cos_sin_cache, angles)):
        for name, x in base.items():
            if not torch.is_tensor(x) or not x.is_floating_point():
                continue
            args = dict(base, **{name: grad(*x.shape, dtype=x.dtype)})
            with pytest.raises(ValueError, match="records no graph"):
                fn(**args)
            with torch.no_grad(), pytest.raises(ValueError, match="GPU only"):
                fn(**args)
