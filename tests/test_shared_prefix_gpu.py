"""Attention of a batch that shares prefixes, against the formula in 64 bits."""
import pytest
import torch

from shared_prefix_tools import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cretif_b200.csrc import ops
    ops.lib()
    return ops


@pytest.fixture(autouse=True)
def no_fault(ops):
    yield
    assert int(ops.fault_word("cuda").item()) == 0


HEADS = [(9, 3, 64), (15, 5, 64), (4, 4, 64), (16, 2, 128), (3, 1, 32), (4, 2, 16), (10, 5, 80), (12, 1, 48),
         (40, 2, 64), (2, 2, 112)]
TYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_heads(ops, heads, dtype):
    Step([([0, 2, 3, 5], 192), ([1, 4], 64)], own=[0, 5, 63, 64, 65, 130, 40], news=[1, 1, 2, 1, 3, 1, 1],
         nh=heads[0], nkv=heads[1], hd=heads[2], dtype=dtype, seed=1).check(ops)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("batch", [1, 2, 3, 7, 21, 43, 64, 130])
def test_batches_on_one_prefix(ops, batch, dtype):
    Step([(list(range(batch)), 256)], own=[(17 * b) % 90 for b in range(batch)], news=[1] * batch, nh=9, nkv=3,
         hd=64, dtype=dtype, seed=batch).check(ops)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 2, 5, 6, 16, 33, 70])
def test_new_tokens(ops, new, dtype):
    """One token, drafts, and more than a tile of them; each sees the ones before it alone."""
    Step([([0, 1, 2], 128)], own=[0, 31, 60], news=[new, 1, max(1, new - 1)], nh=6, nkv=2, hd=64, dtype=dtype,
         seed=new).check(ops)


@pytest.mark.parametrize("own", [0, 1, 62, 63, 64, 127, 128, 300, 1000])
def test_own_keys(ops, own):
    Step([([0, 1], 64)], own=[own, 0], news=[1, 1], nh=9, nkv=3, hd=64, dtype=torch.bfloat16, seed=own).check(ops)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("prefix", [0, 64, 128, 192, 1024, 6400])
def test_prefixes(ops, prefix, dtype):
    Step([([0, 1, 3], prefix)], own=[3, 0, 200, 64], news=[1, 2, 1, 1], nh=8, nkv=4, hd=64, dtype=dtype,
         seed=prefix).check(ops)


@pytest.mark.parametrize("hd", [64, 112])
@pytest.mark.parametrize("batch", [18, 38, 80, 320])
def test_many_rows_a_sequence(ops, batch, hd):
    # (18 x 4 items of 16 rows are fewer than the SMs, 38 x 4 more, 80 x 4 and 320 x 4 take narrower steps)
    s = Step([(list(range(batch)), 320)], own=[(37 * b) % 200 for b in range(batch)],
             news=[1 + (b + 2) % 3 for b in range(batch)], nh=20, nkv=4, hd=hd, dtype=torch.bfloat16, seed=24)
    s.check(ops)


def test_nothing_shared(ops):
    Step([], own=[0, 1, 64, 500], news=[1, 4, 1, 2], nh=9, nkv=3, hd=64, dtype=torch.bfloat16, seed=3).check(ops)


@pytest.mark.parametrize("hd", [64, 128])
def test_many_rows_on_several_prefixes(ops, hd):
    """More rows than a tile holds, groups that end inside one, members in any order."""
    groups = [([0, 5, 9, 12, 20, 21, 22, 33], 640), ([1, 2, 3, 4, 6, 7, 8], 1280), ([30, 10], 64), ([32], 320)]
    Step(groups, own=[(7 * b) % 150 for b in range(34)], news=[1 + b % 6 for b in range(34)], nh=16, nkv=2, hd=hd,
         dtype=torch.bfloat16, seed=5).check(ops)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
def test_sink(ops, dtype):
    s = Step([([0, 1, 2], 192)], own=[1, 30, 64], news=[1, 2, 1], nh=6, nkv=2, hd=64, dtype=dtype, seed=8)
    for sink in (torch.randn(6, generator=torch.Generator().manual_seed(1)).cuda(), torch.full((6,), 40.0).cuda(),
                 torch.full((6,), float("-inf")).cuda()):
        s.check(ops, sink=sink)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("spread", [0.0, 6.0, 40.0])
def test_flat_and_sharp_scores(ops, spread, dtype):
    """Scores that are all equal, and scores so far apart that one key takes all."""
    Step([([0, 1, 2, 3], 512)], own=[2, 70, 0, 9], news=[1, 1, 3, 1], nh=9, nkv=3, hd=64, dtype=dtype, seed=9,
         spread=spread).check(ops)


def test_keys_as_values(ops):
    Step([([0, 1, 2], 256)], own=[2, 70, 0], news=[1, 1, 2], nh=8, nkv=1, hd=128, dtype=torch.bfloat16, seed=10,
         shared_values=True).check(ops)


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), 3e38])
def test_what_lies_behind_a_sequence_is_not_looked_at(ops, poison):
    for dtype in TYPES:
        Step([([0, 1], 64)], own=[0, 37], news=[1, 3], nh=4, nkv=2, hd=64, dtype=dtype, seed=11,
             poison=poison).check(ops)


def test_the_same_bits_twice_and_on_another_stream(ops):
    s = Step([(list(range(20)), 2048)], own=[b for b in range(20)], news=[1 + b % 3 for b in range(20)], nh=9, nkv=3,
             hd=64, dtype=torch.bfloat16, seed=12)
    plan = s.plan(ops)
    first = s.run(ops, plan)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        second = s.run(ops, plan)
    stream.synchronize()
    assert torch.equal(first, second)


def test_one_plan_for_later_steps_of_the_same_batch(ops):
    """The plan knows neither positions nor slots: made for the first step it serves the thirtieth."""
    early = Step([([0, 1, 2], 192)], own=[0, 3, 9], news=[1, 1, 1], nh=9, nkv=3, hd=64, dtype=torch.bfloat16, seed=13)
    late = Step([([0, 1, 2], 192)], own=[400, 403, 9], news=[1, 1, 1], nh=9, nkv=3, hd=64, dtype=torch.bfloat16,
                seed=14)
    late.check(ops, plan=early.plan(ops))
    early.check(ops, plan=late.plan(ops))


def test_two_captured_graphs_at_once(ops):
    """Two graphs of one plan, replayed on two streams at the same time, keep their own scratch."""
    steps = [Step([(list(range(8)), 1024)], own=[5 * b for b in range(8)], news=[1 + b % 2 for b in range(8)], nh=9,
                  nkv=3, hd=64, dtype=torch.bfloat16, seed=s) for s in (15, 16)]
    plan = steps[0].plan(ops)
    want = [s.run(ops, plan).clone() for s in steps]
    graphs, outs = [], []
    for s in steps:
        out = torch.full_like(want[0], 7.0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run(ops, plan, out=out)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run(ops, plan, out=out)
        out.fill_(7.0)
        graphs.append(g)
        outs.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert torch.equal(got, w)


def test_many_steps_in_a_row(ops):
    """Steps launched one behind the other without a wait: each reads what the one before it wrote."""
    s = Step([(list(range(6)), 512)], own=[9 * b for b in range(6)], news=[1] * 6, nh=4, nkv=4, hd=64,
             dtype=torch.bfloat16, seed=17)
    plan = s.plan(ops)
    q0 = s.q.clone()

    def chain(wait):
        q, out = q0.clone(), torch.empty_like(q0)
        for _ in range(12):
            ops.attn_shared(q, out, s.kc, s.vc, s.table, s.tok_pos, s.cu, s.seq_slot, plan, s.scale, 64,
                            ops.fault_word("cuda"))
            if wait:
                torch.cuda.synchronize()
            q, out = out, q
        return q
    assert torch.equal(chain(True), chain(False))


def test_bad_pages_set_the_fault_word(ops):
    s = Step([([0, 1], 128)], own=[10, 70], news=[1, 1], nh=4, nkv=2, hd=64, dtype=torch.bfloat16, seed=18, poison=0.0)
    for spoil in ("prefix", "own", "beyond", "slot", "position"):
        table, slot, pos = s.table.clone(), s.seq_slot.clone(), s.tok_pos.clone()
        if spoil == "prefix":
            table[s.slots[0], 1] = -1
        elif spoil == "own":
            table[s.slots[1], 3] = -1
        elif spoil == "beyond":
            table[s.slots[1], 2] = 10 ** 6
        elif spoil == "slot":
            slot[1] = 50
        else:
            pos[0] = 100
        fault = torch.zeros(1, dtype=torch.int32, device="cuda")
        for dtype in TYPES:
            fault.zero_()
            plan = ops.shared_prefix_plan(s.groups, s.news, s.starts, 4, 2, 64, dtype, "cuda")
            out = torch.empty((2, 256), dtype=dtype, device="cuda")
            ops.attn_shared(s.q.to(dtype), out, s.kc.to(dtype), s.vc.to(dtype), table, pos, s.cu, slot, plan, s.scale,
                            64, fault)
            assert int(fault.item()) == 4, spoil


def test_a_plan_made_on_another_stream(ops):
    s = Step([([0, 1, 2], 640)], own=[10, 70, 0], news=[2, 1, 1], nh=4, nkv=2, hd=64, dtype=torch.bfloat16, seed=22,
             poison=0.0)
    want, side = s.check(ops), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                      # (the plan's copy waits behind it)
        plan = s.plan(ops)
    got = s.run(ops, plan)
    del plan                                               # its memory is not the side stream's again before
    with torch.cuda.stream(side):
        for _ in range(8):
            s.plan(ops).data.fill_(0)
    assert torch.equal(got, want)


def test_no_plan_within_a_capture(ops):
    s = Step([([0, 1], 128)], own=[10, 70], news=[1, 1], nh=4, nkv=2, hd=64, dtype=torch.bfloat16, seed=23)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.zeros(4, device="cuda")                      # (a capture of nothing at all warns)
        with pytest.raises(ops.KernelError, match="before a capture"):
            s.plan(ops)


def test_two_threads_with_heads_of_other_sizes(ops):
    # (the kernels' shared memory goes by the head size)
    import threading
    steps = [Step([([0, 1, 2], 320)], own=[10, 70, 0], news=[2, 1, 1], nh=4, nkv=2, hd=hd, dtype=dtype, seed=21,
                  poison=0.0) for hd in (16, 64, 80, 128) for dtype in TYPES]
    want = [s.check(ops) for s in steps]
    bad = []

    def work(order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    for i in order:
                        if not torch.equal(steps[i].run(ops), want[i]):
                            bad.append(i)
        except Exception as e:                             # (a thread's error would be lost)
            bad.append(repr(e))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(list(range(8))[::d],)) for d in (1, -1)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not bad


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f32"])
def test_a_table_that_is_a_view_ends_where_the_view_does(ops, dtype):
    s = Step([([0, 1], 128)], own=[10, 70], news=[1, 2], nh=4, nkv=2, hd=64, dtype=dtype, seed=20, poison=0.0)
    width = s.table.shape[1]
    wide = torch.zeros((s.table.shape[0], 3 * width), dtype=torch.int32, device="cuda")   # (block 0 beside it)
    wide[:, width:2 * width] = s.table
    whole = s.check(ops)
    s.table = wide[:, width:2 * width]
    assert torch.equal(s.check(ops), whole)
    plan, fault = s.plan(ops), torch.zeros(1, dtype=torch.int32, device="cuda")
    pos = s.tok_pos.clone()
    for at in (64 * width, 128 * width - 1, 2 ** 31 - 257, 2 ** 31 - 1):
        s.tok_pos = pos.clone()
        s.tok_pos[0] = at
        out = s.run(ops, plan, fault=fault.zero_())
        assert int(fault.item()) == 4, at
        assert torch.equal(out[1:], whole[1:])             # (the other sequence's tokens)
    s.tok_pos = pos


def test_refusals(ops):
    s = Step([([0, 1], 128)], own=[10, 70], news=[1, 1], nh=4, nkv=2, hd=64, dtype=torch.bfloat16, seed=19)
    plan = s.plan(ops)
    good = dict(q=s.q, out=torch.empty((2, 256), dtype=torch.bfloat16, device="cuda"), kc=s.kc, vc=s.vc, table=s.table,
                tok_pos=s.tok_pos, cu_seqlens=s.cu, seq_slot=s.seq_slot, plan=plan, scale=s.scale, block_tokens=64,
                fault=ops.fault_word("cuda"))
    ops.attn_shared(**good)
    bad = [dict(q=s.q.float()), dict(q=s.q[:1]), dict(q=s.q[:, :64]), dict(q=s.q.t().contiguous().t()),
           dict(out=good["out"][:, :128]), dict(kc=s.kc[:, :1]), dict(vc=s.vc[:-1]), dict(kc=s.kc.transpose(0, 1)),
           dict(table=s.table[:, :1]), dict(table=s.table.long()), dict(tok_pos=s.tok_pos[:1]),
           dict(cu_seqlens=s.cu[:2]), dict(seq_slot=s.seq_slot[:1]), dict(block_tokens=32), dict(scale=0.0),
           dict(scale=float("nan")), dict(sink=torch.zeros(3, device="cuda")), dict(sink=torch.zeros(4)),
           dict(fault=torch.zeros(1, dtype=torch.int32)), dict(tok_pos=s.tok_pos.cpu())]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.attn_shared(**{**good, **change})
    torch.cuda.synchronize()
