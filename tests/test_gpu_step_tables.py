"""Step tables built on the GPU against a request-by-request loop on the host: integers, so equality."""
import pytest
import torch

from xllm_amd import ops

pytestmark = pytest.mark.gpu


def loop_reference(kv, new, table, free, bs, budget, head):
    """What a host scheduler does, one request after the other."""
    B, W = len(kv), table.shape[1]
    out, seq, cu, indptr, pos, slots, lost = table.clone(), [], [0], [0], [], [], 0
    nxt = min(max(head, 0), len(free))
    for b in range(B):
        k = max(kv[b], 0)
        n = min(max(new[b], 0), budget - cu[-1])
        old = min(-(-k // bs), W)
        need = min(-(-(k + n) // bs), W) - old
        got = min(need, len(free) - nxt)
        out[b, old:] = -1
        for j in range(got):
            out[b, old + j] = free[nxt + j]
        nxt += got
        seq.append(k + n)
        cu.append(cu[-1] + n)
        indptr.append(indptr[-1] + got)
        for t in range(k, k + n):
            page = int(out[b, t // bs]) if t // bs < W else -1
            pos.append(t)
            slots.append(page * bs + t % bs if page >= 0 else -1)
            lost += t >= (old + got) * bs
    pos += [0] * (budget - len(pos))
    slots += [-1] * (budget - len(slots))
    i32 = torch.int32
    return ops.StepTables(out, torch.tensor(seq, dtype=i32), torch.tensor(cu, dtype=i32),
                          torch.tensor(pos, dtype=torch.int64), torch.tensor(slots, dtype=i32),
                          torch.tensor(indptr, dtype=i32), torch.tensor([cu[-1], nxt, lost], dtype=i32))


def assert_tables_equal(got, want):
    for f in ops.StepTables.__dataclass_fields__:
        g, w = getattr(got, f).cpu(), getattr(want, f)
        assert g.dtype == w.dtype and torch.equal(g, w), f"{f}: {g} != {w}"


def make(B, bs, kv_hi, new_hi, seed, extra=2, free=None, kv=None, new=None):
    gen = torch.Generator().manual_seed(seed)
    kv = kv or torch.randint(0, kv_hi + 1, (B,), generator=gen).tolist()
    new = new or torch.randint(0, new_hi + 1, (B,), generator=gen).tolist()
    W = -(-(max(kv) + max(new)) // bs) + extra
    pages = [-(-k // bs) for k in kv]
    pool = sum(pages) + sum(-(-n // bs) + 1 for n in new) + 5
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    table, at = torch.zeros(B, W, dtype=torch.int32), 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    left = order[at:] if free is None else order[at:at + free]
    return kv, new, table, left.contiguous()


def call(kv, new, table, free, bs, budget, head=None, **kw):
    dev = "cuda:0"
    i32 = torch.int32
    return ops.build_step_tables(torch.tensor(kv, dtype=i32, device=dev), torch.tensor(new, dtype=i32, device=dev),
                                 table.to(dev), free.to(dev), bs, budget,
                                 None if head is None else torch.tensor([head], dtype=i32, device=dev), **kw)


@pytest.mark.parametrize("B,bs,kv_hi,new_hi,budget", [
    (1, 16, 0, 1, 1), (1, 16, 100, 0, 4), (3, 1, 9, 4, 16), (5, 24, 200, 50, 400), (64, 16, 300, 1, 64),
    (63, 16, 64, 33, 1100), (65, 128, 700, 300, 12000), (257, 16, 40, 9, 1500), (1025, 8, 33, 3, 2500),
    (4100, 16, 20, 2, 5000)])
def test_against_the_loop(B, bs, kv_hi, new_hi, budget):
    kv, new, table, free = make(B, bs, kv_hi, new_hi, seed=B + bs)
    got = call(kv, new, table, free, bs, budget)
    assert_tables_equal(got, loop_reference(kv, new, table, free.tolist(), bs, budget, 0))


@pytest.mark.parametrize("B", [255, 256, 258, 511, 512, 513, 1023, 1024, 1026, 2047, 2048, 2050, 4095, 4096])
@pytest.mark.parametrize("short", [False, True])
def test_batches_around_the_ends_of_a_workgroup(B, short):
    """Where a thread takes one request more, and token counts around whole workgroups; short: budget and pages run out."""
    kv, new, table, free = make(B, 16, 60, 3, seed=B, extra=1)
    budget = sum(new) - 257 if short else sum(new) + 255
    if short:
        free = free[:B // 4].contiguous()
    got = call(kv, new, table, free, 16, budget)
    assert_tables_equal(got, loop_reference(kv, new, table, free.tolist(), 16, budget, 0))


@pytest.mark.parametrize("case", ["budget", "no budget", "free list", "empty free list", "width", "head", "head beyond",
                                  "negative lengths", "hole", "wide"])
def test_what_runs_out(case):
    bs, budget, head = 16, 300, None
    kv, new, table, free = make(20, bs, 100, 40, seed=7)
    if case == "budget":
        budget = 123
    elif case == "no budget":
        budget = 0
    elif case == "free list":
        free = free[:9].contiguous()
    elif case == "empty free list":
        free = free[:0].contiguous()
    elif case == "width":
        table = table[:, :4].contiguous()
    elif case == "head":
        head = 5
    elif case == "head beyond":
        head = free.numel() + 3
    elif case == "negative lengths":
        kv[3], new[5], new[6] = -7, -1, -2147483648
        budget = 999
    elif case == "hole":
        b = max(range(20), key=lambda i: kv[i] % bs)
        table[b, kv[b] // bs] = -1
        new[b] = max(new[b], 1)
        budget = 2000
    elif case == "wide":   # rows longer than a workgroup's share of the table
        table = torch.cat([table, torch.full((20, 2500), 9, dtype=torch.int32)], 1)
    got = call(kv, new, table, free, bs, budget, head)
    want = loop_reference(kv, new, table, free.tolist(), bs, budget, head or 0)
    assert_tables_equal(got, want)
    if case in ("free list", "empty free list", "width", "head beyond"):
        assert int(want.counters[2]) > 0


def test_lengths_at_the_ends_of_their_range():
    """A context of 2^31 - 1 tokens and a request for as many: sums and pages stay in range."""
    top = 2 ** 31 - 1
    kv, new = [top, 3, 0], [5, top, top]
    table = torch.arange(12, dtype=torch.int32).view(3, 4)
    free = torch.arange(100, 140, dtype=torch.int32)
    got = call(kv, new, table, free, 2 ** 29, 16)
    assert got.q_cu_seq_lens.tolist() == [0, 5, 16, 16] and got.seq_lens.tolist() == [top, 14, 0]
    assert got.position_ids.tolist() == [top + i for i in range(5)] + list(range(3, 14))
    # request 0's first token is the last one of page 3, 3 * 2^29 + 2^29 - 1 = 2^31 - 1, and its next ones lie behind the
    # table; request 1's page 4 times 2^29 passes 31 bits
    assert got.slot_mapping.tolist() == [top] + [-1] * 15
    assert got.block_table.tolist()[0] == [0, 1, 2, 3] and got.counters.tolist()[0] == 16


def test_in_place_keeps_the_pages_and_the_rows_around():
    kv, new, table, free = make(33, 16, 90, 30, seed=3)
    wide = torch.full((33, table.shape[1] + 7), 77, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    dev_wide = wide.cuda()
    view = dev_wide[:, 2:2 + table.shape[1]]
    B, T = 33, 700
    i32 = dict(dtype=torch.int32, device="cuda")
    out = ops.StepTables(view, torch.empty(B, **i32), torch.empty(B + 1, **i32),
                         torch.empty(T, dtype=torch.int64, device="cuda"), torch.empty(T, **i32), torch.empty(B + 1, **i32),
                         torch.empty(3, **i32))
    for _ in range(2):   # (the same call again finds the same pages)
        got = ops.build_step_tables(torch.tensor(kv, **i32), torch.tensor(new, **i32), view, free.cuda(), 16, T, out=out)
        assert got is out
        assert_tables_equal(got, loop_reference(kv, new, table, free.tolist(), 16, T, 0))
    after = dev_wide.cpu()
    assert (after[:, :2] == 77).all() and (after[:, 2 + table.shape[1]:] == 77).all()


def test_captured_steps_follow_their_inputs():
    """One captured step replayed over several: the lengths and the free head are fed back between the replays."""
    B, bs, W, T = 9, 4, 12, 16
    i32 = dict(dtype=torch.int32, device="cuda")
    kv, new, head = torch.zeros(B, **i32), torch.ones(B, **i32), torch.zeros(1, **i32)
    table, free = torch.full((B, W), -1, **i32), torch.randperm(64, device="cuda").to(torch.int32)
    out = ops.StepTables(table, torch.empty(B, **i32), torch.empty(B + 1, **i32),
                         torch.empty(T, dtype=torch.int64, device="cuda"), torch.empty(T, **i32), torch.empty(B + 1, **i32),
                         torch.empty(3, **i32))
    ops.build_step_tables(kv, new, table, free, bs, T, head, out=out)
    table.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.build_step_tables(kv, new, table, free, bs, T, head, out=out)
        kv.copy_(out.seq_lens)
        head.copy_(out.counters[1:2])
    ref_kv, ref_table, ref_head = [0] * B, torch.full((B, W), -1, dtype=torch.int32), 0
    gen = torch.Generator().manual_seed(1)
    for step in range(12):
        n = torch.randint(0, 3, (B,), generator=gen).tolist()
        new.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = loop_reference(ref_kv, n, ref_table, free.tolist(), bs, T, ref_head)
        assert_tables_equal(out, want)
        ref_kv, ref_table, ref_head = want.seq_lens.tolist(), want.block_table, int(want.counters[1])
        torch.empty(1 << 16, device="cuda").fill_(step)


def test_another_stream():
    kv, new, table, free = make(40, 16, 90, 30, seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(kv, new, table, free, 16, 800)
    side.synchronize()
    assert_tables_equal(got, loop_reference(kv, new, table, free.tolist(), 16, 800, 0))


def test_no_requests():
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ops.build_step_tables(torch.empty(0, **i32), torch.empty(0, **i32), torch.empty(0, 4, **i32), torch.arange(5, **i32),
                                16, 3, torch.tensor([2], **i32))
    assert got.counters.tolist() == [0, 2, 0] and got.slot_mapping.tolist() == [-1] * 3 and got.position_ids.tolist() == [0] * 3


@pytest.mark.parametrize("B", [0, 3])
def test_a_free_head_inside_the_results_is_refused(B):
    """The next step's head is counters[1]; handed over as a view of the very counters that the call writes it would be lost."""
    i32 = dict(dtype=torch.int32, device="cuda")
    kv, new, table, free = torch.zeros(B, **i32), torch.ones(B, **i32), torch.zeros(B, 4, **i32), torch.arange(9, **i32)
    out = ops.build_step_tables(kv, new, table, free, 16, 6, torch.tensor([2], **i32))
    head = int(out.counters[1])
    assert head == 2 + B
    for view in (out.counters[1:2], out.q_cu_seq_lens[:1], out.new_page_indptr[:1], out.slot_mapping[5:6]):
        with pytest.raises(ValueError, match="overlaps"):
            ops.build_step_tables(kv, new, table, free, 16, 6, view, out=out)
    assert int(out.counters[1]) == head
    ops.build_step_tables(kv, new, table, free, 16, 6, out.counters[1:2].clone(), out=out)
    assert int(out.counters[1]) == head + B


def test_refusals():
    i32 = dict(dtype=torch.int32, device="cuda")
    kv, new, table, free = torch.zeros(4, **i32), torch.ones(4, **i32), torch.zeros(4, 3, **i32), torch.arange(9, **i32)
    good = ops.build_step_tables(kv, new, table, free, 16, 8)
    bad = [(kv.long(), new, table, free, 16, 8), (kv, new[:3], table, free, 16, 8), (kv, new, table.t(), free, 16, 8),
           (kv, new, table, free, 0, 8), (kv, new, table, free, 16, -1), (kv, new, table[:3], free, 16, 8),
           (kv, new, table, free.view(3, 3), 16, 8), (kv, new, table[:1].expand(4, 3), free, 16, 8)]
    for args in bad:
        with pytest.raises((ValueError, TypeError)):
            ops.build_step_tables(*args)
    with pytest.raises(ValueError):
        ops.build_step_tables(kv.cpu(), new, table, free, 16, 8)
    for field, value in (("seq_lens", kv), ("slot_mapping", good.slot_mapping[:7]), ("counters", good.counters.long()),
                         ("block_table", good.block_table[:, :2]), ("new_page_indptr", good.q_cu_seq_lens)):
        args = {f: getattr(good, f) for f in ops.StepTables.__dataclass_fields__}
        args[field] = value
        with pytest.raises(ValueError):
            ops.build_step_tables(kv, new, table, free, 16, 8, out=ops.StepTables(**args))
