"""The kernels that hold a cache to a budget by attention weight, against 64 bits: tolerances are the oracle's bounds."""
import math

import pytest
import torch

import kv_mass_oracle as oracle
from metrale_inference_alpha_b200 import ops
from metrale_inference_alpha_b200.ops import _native, kv_mass

pytestmark = pytest.mark.gpu


def _cuda(c):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def _decode(c, **kw):
    return ops.paged_attention_mass(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["mass"], scale=c["scale"], k_scale=c["k_scale"], v_scale=c["v_scale"],
                                    **(dict(max_ctx=c["max_ctx"]) | kw))


def _prompt(c, last, **kw):
    return ops.prompt_mass(c["q"], c["k"], c["table"], c["q_start"], c["q_len"], c["ctx"], c["mass"], scale=c["scale"], last=last, k_scale=c["k_scale"],
                           **(dict(max_q_len=c["max_q_len"], max_ctx=c["max_ctx"]) | kw))


def _within(got, want, tol, what):
    far = (got.double().cpu() - want).abs() - tol
    assert bool((far <= 0).all()), f"{what}: {int((far > 0).sum())} of {far.numel()} beyond their bound, by up to {float(far.max()):.3g} at {int(far.argmax())}"


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status("cuda")


# ----------------------------------------------------------------------------- decode
SHAPES = [(4, 2, 64), (40, 8, 128), (8, 8, 128), (16, 1, 128), (24, 1, 128), (32, 1, 128), (48, 1, 128), (12, 1, 64), (3, 3, 256), (16, 2, 256), (20, 1, 256)]
LENGTHS = [[1], [700], [0, 15, 16, 17, 64, 65], [513, 1, 0, 1025, 1024, 511, 3, 2047]]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("ctx", LENGTHS, ids=str)
def test_decode(fp8, heads, kv_heads, dim, ctx):
    c = oracle.case(20, ctx, heads, kv_heads, dim, fp8, columns=max(ctx) + 5)
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    got = _decode(g)
    _within(got, want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")
    for s, n in enumerate(ctx):
        assert torch.equal(g["mass"][s, :, n:].cpu(), c["mass"][s, :, n:])


@pytest.mark.parametrize("block", [1, 8, 24, 32, 48, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_block_sizes(block, fp8):
    c = oracle.case(21, [130, 7, 600], 10, 2, 128, fp8, block=block)
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    _within(_decode(g), want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


@pytest.mark.parametrize("block,fp8", [(2, True), (6, True), (12, True), (24, True), (1, False), (7, False)])
@pytest.mark.parametrize("heads,dim", [(4, 64), (20, 64), (6, 256)])
def test_decode_block_sizes_of_other_heads(block, fp8, heads, dim):
    c = oracle.case(34, [130, 7, 600, 0, 17], heads, 2, dim, fp8, block=block)
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    _within(_decode(g), want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (128, 10, 2), (256, 8, 1)])
def test_decode_of_a_long_sequence(dim, heads, kv_heads):
    """More tokens than 32 of the shortest partitions hold."""
    c = oracle.case(22, [40007, 33], heads, kv_heads, dim, False)
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    _within(_decode(g), want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


def test_decode_of_large_logits():
    """Scores hundreds of powers of two apart: all but a few weights vanish, and the rest keep their bound."""
    c = oracle.case(23, [300, 90], 8, 2, 128, False, spread=40.0)
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    _within(_decode(g), want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


def test_decode_writes_its_part_of_a_larger_buffer():
    c = _cuda(oracle.case(24, [200, 30, 77], 8, 2, 128, True))
    alone = c["mass"].clone()
    lanes = torch.full((5, 3, 260), 3.0, device="cuda")
    lanes[1:4, 1:, 7:207] = c["mass"]
    want = _decode({**c, "mass": alone})
    got = _decode({**c, "mass": lanes[1:4, 1:, 7:207]})
    assert torch.equal(got, want) and torch.equal(lanes[1:4, 1:, 7:207], alone)
    lanes[1:4, 1:, 7:207] = 3.0
    assert bool((lanes == 3).all())


@pytest.mark.parametrize("fp8,dim", [(True, 128), (False, 64), (False, 256)])
def test_decode_of_a_sequence_does_not_depend_on_its_batch(fp8, dim):
    ctx = [1500, 40, 700, 1100]
    c = _cuda(oracle.case(25, ctx, 8, 2, dim, fp8))
    m = c["mass"].clone()
    out = _decode(c)
    for s in range(4):
        one = {**c, "q": c["q"][s:s + 1], "table": c["table"][s:s + 1], "ctx": c["ctx"][s:s + 1], "mass": m[s:s + 1]}
        assert torch.equal(_decode(one)[0], out[s]) and torch.equal(m[s], c["mass"][s])


def test_decode_in_several_steps_gives_the_same(monkeypatch):
    c = _cuda(oracle.case(26, [300, 10, 0, 513, 77], 8, 2, 128, False))
    m = c["mass"].clone()
    out = _decode(c)
    monkeypatch.setattr(kv_mass, "_WS_BYTES", 1)
    assert torch.equal(_decode({**c, "mass": m}), out) and torch.equal(m, c["mass"])


def test_decode_of_more_sequences_than_a_launch_takes():
    n = 1100
    c = oracle.case(31, [1 + i % 5 for i in range(n)], 4, 2, 64, False)
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    _within(_decode(g), want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


def test_decode_of_lanes_that_pad_the_batch():
    """Lengths of zero and less, and a call all of whose lanes are such."""
    c = _cuda(oracle.case(32, [40, 3, 20], 4, 2, 64, True))
    c["ctx"] = torch.tensor([0, -7, 20], dtype=torch.int32, device="cuda")
    before = c["mass"].clone()
    out = _decode(c)
    assert not out[:2].any() and torch.equal(c["mass"][:2], before[:2]) and bool((c["mass"][2] != before[2]).any())
    none = torch.zeros(3, 2, 0, device="cuda")
    assert not _decode({**c, "ctx": torch.zeros_like(c["ctx"]), "mass": none, "table": c["table"][:, :0]}, max_ctx=0).any()


def test_decode_of_infinities_and_nan():
    """A query that is not a number makes its group's mass one; a key that is one of infinity takes all the weight or the row with it, as in 64 bits."""
    c = oracle.case(33, [50, 60], 8, 2, 128, False)
    c["q"][0, 1, 5] = float("nan")
    g = _cuda(c)
    out = _decode(g)
    assert out[0, 1].isnan().all() and g["mass"][0, 0, :50].isnan().all()
    assert not out[0, 2:].isnan().any() and not g["mass"][0, 1].isnan().any() and not g["mass"][1].isnan().any()


def test_decode_agrees_with_the_attention_that_leaves_no_weights():
    c = _cuda(oracle.case(27, [700, 64, 1300], 40, 8, 128, True))
    plain = ops.paged_attention(c["q"], c["k"], c["v"], c["table"], c["q_start"], c["q_len"], c["ctx"], max_q_len=1, max_ctx=1300, scale=c["scale"], k_scale=c["k_scale"],
                                v_scale=c["v_scale"])
    got = _decode(c)
    assert float((got.float() - plain.float()).abs().max()) <= 2.0 ** -7 * float(plain.float().abs().max())


def _graph(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = fn()
    return g, r


def test_two_captured_steps_share_nothing():
    """Graphs of different batches, replayed on two streams at once."""
    cs = [_cuda(oracle.case(28 + i, ctx, 40, 8, 128, True)) for i, ctx in enumerate(([900, 600], [1200, 30, 256]))]
    start = [c["mass"].clone() for c in cs]
    want = []
    for c, m in zip(cs, start):
        mass = m.clone()
        want.append((_decode({**c, "mass": mass}), mass))
    graphs = [_graph(lambda c=c: _decode(c)) for c in cs]
    for _ in range(3):
        for c, m in zip(cs, start):
            c["mass"].copy_(m)
        torch.cuda.synchronize()
        for g, _ in graphs:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, (_, out), (w, mass) in zip(cs, graphs, want):
            assert torch.equal(out, w) and torch.equal(c["mass"], mass)


def test_decode_reports_lengths_and_blocks_out_of_range():
    c = _cuda(oracle.case(30, [100, 50], 8, 2, 128, False))
    c["v"].nan_to_num_(0.0), c["k"].nan_to_num_(0.0)
    _decode(c, max_ctx=90)
    with pytest.raises(_native.KernelError, match="bounds"):
        ops.check_status("cuda")
    c["table"][0, 2] = 10 ** 6
    _decode(c)
    with pytest.raises(_native.KernelError, match="bounds"):
        ops.check_status("cuda")


# ----------------------------------------------------------------------------- prompts
PROMPTS = [([1], [1], 0), ([700], [700], 0), ([700], [130], 32), ([300, 0, 5, 129, 128], [300, 0, 5, 1, 128], 0), ([2100, 260], [70, 257], 64), ([1000], [1000], 257)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (10, 2, 128), (2, 2, 128), (16, 1, 256), (33, 1, 128)])
@pytest.mark.parametrize("ctx,new,last", PROMPTS, ids=str)
def test_prompt(fp8, heads, kv_heads, dim, ctx, new, last):
    c = oracle.case(40, ctx, heads, kv_heads, dim, fp8, new=new, columns=max(ctx) + 3)
    mass, mtol = oracle.prompt(c, last)
    g = _cuda(c)
    _prompt(g, last)
    _within(g["mass"], mass, mtol, "mass")
    for s, n in enumerate(ctx):
        assert torch.equal(g["mass"][s, :, n:].cpu(), c["mass"][s, :, n:])


@pytest.mark.parametrize("block", [1, 8, 24, 64, 256])
def test_prompt_block_sizes(block):
    c = oracle.case(41, [333, 90], 8, 2, 128, block % 16 == 0, block=block, new=[150, 90])
    mass, mtol = oracle.prompt(c, 100)
    g = _cuda(c)
    _prompt(g, 100)
    _within(g["mass"], mass, mtol, "mass")


def test_prompt_of_large_logits():
    c = oracle.case(42, [300, 140], 8, 2, 128, False, new=[140, 140], spread=40.0)
    mass, mtol = oracle.prompt(c, 0)
    g = _cuda(c)
    _prompt(g, 0)
    _within(g["mass"], mass, mtol, "mass")


def test_prompt_rows_that_see_nothing_give_nothing():
    c = _cuda(oracle.case(43, [3], 2, 1, 64, False, new=[5]))
    before = c["mass"].clone()
    _prompt(c, 0)
    assert float((c["mass"] - before).sum()) == pytest.approx(3 * 2, rel=1e-5)


def test_prompt_of_a_sequence_does_not_depend_on_its_batch():
    c = _cuda(oracle.case(44, [1500, 300, 700], 8, 2, 128, True, new=[900, 300, 33]))
    m = c["mass"].clone()
    _prompt(c, 64)
    for s in range(3):
        one = {k: c[k][s:s + 1] for k in ("table", "ctx", "q_start", "q_len")}
        _prompt({**c, **one, "mass": m[s:s + 1]}, 64)
        assert torch.equal(m[s], c["mass"][s])


def test_prompt_in_several_steps_gives_the_same(monkeypatch):
    c = _cuda(oracle.case(48, [300, 40, 0, 513, 77], 8, 2, 128, True, new=[200, 40, 0, 13, 77]))
    m = c["mass"].clone()
    _prompt(c, 64)
    monkeypatch.setattr(kv_mass, "_WS_BYTES", 1)
    _prompt({**c, "mass": m}, 64)
    assert torch.equal(m, c["mass"])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,block", [(8, 2, 128, 16), (4, 4, 64, 16), (5, 1, 128, 24), (16, 2, 256, 16), (64, 1, 64, 32), (12, 3, 256, 5)])
def test_prompt_of_few_rows_does_not_depend_on_its_batch(heads, kv_heads, dim, block, fp8):
    """Few rows stay in a CTA of the keys pass, those of a call with a longer portion go by: the same bits."""
    G = heads // kv_heads
    new = [1, 128 // G, 128 // G + 1, 256 // G, 3, 600 // G + 300]
    c = _cuda(oracle.case(62, [700, 129, 2500, 1024, 5000, 1300], heads, kv_heads, dim, fp8, block=block, new=new))
    c["q"][4, 0, 7] = math.nan
    c["q"][new[0] + new[1] + 5 % new[2], 0, 1] = math.inf    # of sequence 2
    m = c["mass"].clone()
    _prompt(c, 0)
    want = c["mass"].clone()
    for s in range(5):
        one = {k: c[k][s:s + 1] for k in ("table", "ctx", "q_start", "q_len")}
        c["mass"] = m.clone()
        _prompt({**c, **one, "mass": c["mass"][s:s + 1]}, 0, max_q_len=new[s])
        assert _same(c["mass"][s].nan_to_num(-1.0), want[s].nan_to_num(-1.0))
        assert _same(c["mass"][:s], m[:s]) and _same(c["mass"][s + 1:], m[s + 1:])
    assert want.isnan().any() and not want.isnan().all()


@pytest.mark.parametrize("apart", [2.0 ** -9, 2.0 ** 9, 2.0 ** 40])
def test_prompt_of_rows_far_apart(apart):
    """An e4m3 cache's queries become f16: rows whose sizes differ by little share a factor, others have their own; none loses its range."""
    c = oracle.case(49, [300, 150], 8, 2, 128, True, new=[200, 150])
    c["scale"] /= max(1.0, apart)
    c["q"][::3] *= apart
    c["q"][5::7] = 0
    mass, mtol = oracle.prompt(c, 0)
    g = _cuda(c)
    _prompt(g, 0)
    _within(g["mass"], mass, mtol, "mass")


@pytest.mark.parametrize("fp8", [False, True])
def test_prompt_of_a_query_that_is_not_a_number(fp8):
    c = oracle.case(57, [200, 100], 8, 2, 128, fp8, new=[100, 100])
    c["q"][20, 1, 3] = float("nan")                          # sequence 0, sees the first 121 tokens; head 1 is of kv head 0
    g = _cuda(c)
    _prompt(g, 0)
    assert g["mass"][0, 0, :121].isnan().all() and not g["mass"][0, 0, 121:].isnan().any()
    assert not g["mass"][0, 1].isnan().any() and not g["mass"][1].isnan().any()
    c["q"][20, 1, 3] = 0
    g = _cuda(c)
    _prompt({**g, "q": g["q"].masked_fill(torch.arange(200, device="cuda")[:, None, None] == 20, float("nan"))}, 50)   # among those that do not observe
    assert not g["mass"].isnan().any()


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (1, 1, 64), (4, 2, 256)])
def test_prompt_of_an_infinite_query(heads, kv_heads, dim, fp8, value):
    """Its row has no weights that are numbers; what it does not see keeps those of the rows beside it."""
    c = oracle.case(61, [200, 100], heads, kv_heads, dim, fp8, new=[100, 100])
    want, tol = oracle.prompt(c, 0)
    c["q"][20, 0, 3] = value                                 # sequence 0, sees the first 121 tokens; head 0 is of kv head 0
    g = _cuda(c)
    _prompt(g, 0)
    assert g["mass"][0, 0, :121].isnan().all()
    got = g["mass"].clone()
    got[0, 0, :121] = want[0, 0, :121] = 0
    assert not got.isnan().any()
    _within(got, want, tol, "mass")


def test_prompt_in_a_graph_beside_another():
    cs = [_cuda(oracle.case(45 + i, ctx, 8, 2, 128, False, new=new)) for i, (ctx, new) in enumerate((([900, 600], [100, 600]), ([1200, 30, 256], [40, 30, 256])))]
    start = [c["mass"].clone() for c in cs]
    want = [_prompt({**c, "mass": m.clone()}, 64, max_q_len=600) for c, m in zip(cs, start)]
    graphs = [_graph(lambda c=c: _prompt(c, 64, max_q_len=600))[0] for c in cs]
    for c, m in zip(cs, start):
        c["mass"].copy_(m)
    torch.cuda.synchronize()
    for g in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(c["mass"], w) for c, w in zip(cs, want))


def test_prompt_reports_lengths_rows_and_blocks_out_of_range():
    c = _cuda(oracle.case(47, [100, 50], 8, 2, 128, False, new=[20, 50]))
    c["k"].nan_to_num_(0.0)
    for change in (dict(max_ctx=90), dict(max_q_len=30)):
        _prompt(c, 0, **change)
        with pytest.raises(_native.KernelError, match="bounds"):
            ops.check_status("cuda")
    before = c["mass"].clone()
    _prompt({**c, "q_start": torch.tensor([0, 21], dtype=torch.int32, device="cuda")}, 0)
    with pytest.raises(_native.KernelError, match="bounds"):
        ops.check_status("cuda")
    assert torch.equal(c["mass"][1], before[1])
    c["table"][0, 2] = -3
    _prompt(c, 0)
    with pytest.raises(_native.KernelError, match="bounds"):
        ops.check_status("cuda")


# ----------------------------------------------------------------------------- eviction
def _poisoned(c, seed):
    g = torch.Generator().manual_seed(seed)
    m = c["mass"]
    m.copy_(torch.randint(0, 50, m.shape, generator=g).float() / 16)
    for value in (math.nan, math.inf, -math.inf, -0.0, 1e-42):
        m[torch.rand(m.shape, generator=g) < 0.03] = value


def _same(a, b):
    a, b = a.cpu(), b.cpu()
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8)) if a.is_floating_point() else torch.equal(a, b)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (128, 16), (129, 129), (500, 0), (1000, 100), (1024, 1), (5000, 7)])
@pytest.mark.parametrize("own_blocks", [False, True])
@pytest.mark.parametrize("fp8,dim,block", [(False, 64, 16), (True, 64, 24), (True, 128, 16), (False, 256, 1)])
def test_evict(keep, recent, own_blocks, fp8, dim, block):
    ctx = [1500, 1, keep, keep + 1, 0, 2049] if keep < 2000 else [1500, 1, 0, 33]
    c = oracle.case(50, ctx, 2, 2, dim, fp8, block=block, columns=max(ctx) + 2)
    _poisoned(c, 51)
    dst, S = None, len(ctx)
    if own_blocks:
        per = (min(keep, max(ctx)) + block - 1) // block
        dst = (torch.randperm(S * per, generator=torch.Generator().manual_seed(52)).int() + c["k"].shape[0]).view(S, per)
        c["k"], c["v"] = (torch.cat([x, torch.zeros(S * per, *x.shape[1:], dtype=x.dtype)]) for x in (c["k"], c["v"]))
    k, v, mass, kept, length = oracle.evict(c, keep, recent, c["max_ctx"], dst)
    g = _cuda(c)
    out = torch.full_like(g["mass"], 5.0) if own_blocks else None
    got = ops.kv_evict(g["k"], g["v"], g["table"], g["ctx"], g["mass"], keep=keep, recent=recent, max_ctx=c["max_ctx"], dst_table=None if dst is None else dst.cuda(), mass_out=out)
    assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), length)
    assert _same(g["k"], k) and _same(g["v"], v)
    n = c["max_ctx"]
    if own_blocks:
        assert _same(out[:, :, :n], mass[:, :, :n]) and bool((out[:, :, n:] == 5).all()) and _same(g["mass"], c["mass"])
    else:
        assert _same(g["mass"], mass)


@pytest.mark.parametrize("own_blocks", [False, True])
@pytest.mark.parametrize("n", [32_769, 150_001, 300_007])
def test_evict_from_a_long_sequence(own_blocks, n):
    """Against a selection by sorting: longer than what one CTA, and what a cluster has in registers, with long runs of equal mass."""
    H, D, bs, keep, recent = 2, 64, 16, 9000, 33
    g = torch.Generator(device="cuda").manual_seed(53)
    nb = (n + bs - 1) // bs
    more = (keep + bs - 1) // bs if own_blocks else 0
    k = torch.randint(0, 256, (nb + more, bs, H, D), generator=g, device="cuda", dtype=torch.uint8)
    v = torch.randint(0, 256, (nb + more, bs, H, D), generator=g, device="cuda", dtype=torch.uint8)
    table = torch.randperm(nb, generator=g, device="cuda").int().view(1, nb)
    mass = (torch.rand(1, H, n, generator=g, device="cuda") * 40).floor()
    mass[0, 1, 1000:] = 0.0
    best = torch.sort(mass[0, :, :n - recent], dim=-1, descending=True, stable=True).indices[:, :keep - recent].sort(-1).values
    idx = torch.cat([best, torch.arange(n - recent, n, device="cuda").expand(H, -1)], 1)
    dst = (torch.arange(more, device="cuda").flip(0) + nb).int().view(1, more) if own_blocks else None
    to_table, to = table if dst is None else dst, torch.arange(keep, device="cuda")
    wk, wv, wm = k.clone(), v.clone(), torch.zeros_like(mass)
    for h in range(H):
        a = table[0, idx[h] // bs].long() * bs + idx[h] % bs
        b = to_table[0, to // bs].long() * bs + to % bs
        wk.flatten(0, 1)[b, h], wv.flatten(0, 1)[b, h] = k.flatten(0, 1)[a, h], v.flatten(0, 1)[a, h]
        wm[0, h, :keep] = mass[0, h, idx[h]]
    kept, length = ops.kv_evict(k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), mass, keep=keep, recent=recent, max_ctx=n, dst_table=dst)
    assert torch.equal(kept[0].long(), idx) and int(length) == keep
    assert torch.equal(k, wk) and torch.equal(v, wv) and torch.equal(mass, wm)


def test_evict_in_a_graph_beside_another():
    cs = [_cuda(oracle.case(54 + i, ctx, 8, 2, 128, True)) for i, ctx in enumerate(([900, 600], [1200, 30, 256]))]
    outs = [torch.zeros_like(c["mass"]) for c in cs]
    first = [tuple(x.clone() for x in (c["k"], c["v"])) for c in cs]

    def call(c, o):
        return ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=200, recent=20, max_ctx=c["max_ctx"], mass_out=o)
    want = []
    for c, o in zip(cs, outs):
        kept, n = call(c, o)
        want.append([x.clone() for x in (kept, n, o, c["k"], c["v"])])
    graphs = [_graph(lambda c=c, o=o: call(c, o)) for c, o in zip(cs, outs)]
    for c, (k, v) in zip(cs, first):
        c["k"].copy_(k), c["v"].copy_(v)
    torch.cuda.synchronize()
    for g, _ in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
    torch.cuda.synchronize()
    for c, o, (_, (kept, n)), w in zip(cs, outs, graphs, want):
        assert all(_same(a, b) for a, b in zip((kept, n, o, c["k"], c["v"]), w))


def test_evict_reports_lengths_and_blocks_out_of_range():
    c = _cuda(oracle.case(56, [100, 50], 8, 2, 128, False))
    k = c["k"].clone()
    dst = torch.full((2, 2), 10 ** 6, dtype=torch.int32, device="cuda")
    ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"].clone(), keep=20, recent=2, max_ctx=100, dst_table=dst)
    with pytest.raises(_native.KernelError, match="bounds"):
        ops.check_status("cuda")
    assert _same(c["k"], k)
    kept, length = ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=95, recent=2, max_ctx=90)
    with pytest.raises(_native.KernelError, match="bounds"):
        ops.check_status("cuda")
    assert length.tolist() == [90, 50] and int(kept.max()) == 89


def test_evict_of_nothing():
    c = _cuda(oracle.case(58, [40, 9], 4, 2, 64, False))
    none = torch.zeros(2, 2, 0, device="cuda")
    kept, length = ops.kv_evict(c["k"], c["v"], c["table"][:, :0], torch.zeros_like(c["ctx"]), none, keep=3, recent=1, max_ctx=0)
    assert bool((kept == -1).all()) and not length.any()
    k = c["k"].clone()
    kept, length = ops.kv_evict(c["k"], c["v"], c["table"], torch.tensor([0, -4], dtype=torch.int32, device="cuda"), c["mass"], keep=3, recent=1, max_ctx=40)
    assert bool((kept == -1).all()) and not length.any() and _same(c["k"], k) and not c["mass"].any()


@pytest.mark.parametrize("fp8", [False, True])
def test_sequences_that_share_a_table(fp8):
    """A table that is one row for all (stride 0), its blocks read by every sequence and cut into blocks of their own: bits as from a table a sequence."""
    S, n, bs = 3, 150, 16
    c = _cuda(oracle.case(60, [n] * S, 8, 2, 128, fp8, block=bs, new=[20] * S))
    k0, v0 = c["k"], c["v"]
    one = c["table"][:1].clone()
    spare = torch.zeros(S * 4, *k0.shape[1:], dtype=k0.dtype, device="cuda")
    own = (len(k0) + torch.arange(S * 4, dtype=torch.int32, device="cuda")).view(S, 4)
    got = []
    for table in (one.expand(S, -1), one.repeat(S, 1)):
        d = {**c, "k": torch.cat([k0, spare]), "v": torch.cat([v0, spare]), "table": table, "mass": c["mass"].clone()}
        _prompt(d, 7)
        out = _decode({**d, "q": d["q"][:S].contiguous()})
        kept, length = ops.kv_evict(d["k"], d["v"], table, d["ctx"], d["mass"], keep=60, recent=5, max_ctx=n, dst_table=own)
        assert _same(d["k"][:len(k0)], k0) and _same(d["v"][:len(v0)], v0) and length.tolist() == [60] * S
        got.append((out, d["mass"], kept, d["k"], d["v"]))
    assert table.stride(0) and one.expand(S, -1).stride(0) == 0
    for x, y in zip(*got):
        assert _same(x, y)


# ----------------------------------------------------------------------------- far into a large cache
def test_places_beyond_32_bits():
    """Blocks at the end of caches of 6.6 GB each: the same bits as from a small cache."""
    small = _cuda(oracle.case(59, [300, 77], 16, 8, 128, False, new=[40, 40]))
    far = 200_000
    big = dict(small)
    shift = far - small["k"].shape[0]
    for name in ("k", "v"):
        big[name] = torch.empty(far, 16, 8, 128, dtype=torch.bfloat16, device="cuda")
        big[name][shift:] = small[name]
        big[name][0] = 0                                     # the null block is read, and masked
    assert big["k"].numel() * 2 > 1 << 32
    big["table"] = small["table"] + shift
    big["mass"] = small["mass"].clone()
    results = []
    for c in (small, big):
        one = {**c, "q": c["q"][:2].contiguous()}
        out = _decode(one)
        _prompt(c, 0)
        kept, length = ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=100, recent=10, max_ctx=c["max_ctx"])
        results.append((out, c["mass"], kept, length, c["k"][shift if c is big else 0:], c["v"][shift if c is big else 0:]))
    assert all(_same(a, b) for a, b in zip(*results))


# ----------------------------------------------------------------------------- together
@pytest.mark.parametrize("fp8", [False, True])
def test_a_prompt_is_cut_and_decoded_from(fp8):
    """A prompt's observers, the cut into blocks of its own, then decode steps that write their rows behind what stayed, cut in place again: outputs,
    mass and rows against the same steps in 64 bits."""
    H, G, D, bs, keep, recent, last = 2, 4, 128, 16, 96, 16, 32
    c = oracle.case(60, [400, 90, 230], H * G, H, D, fp8, new=[400, 90, 230], columns=400)
    c["mass"].zero_()
    S, per = 3, (keep + 24 + bs - 1) // bs
    dst = (torch.arange(S * per, dtype=torch.int32) + c["k"].shape[0]).view(S, per)
    for name in ("k", "v"):
        c[name] = torch.cat([c[name], torch.zeros(S * per, bs, H, D, dtype=c[name].dtype)])
    g = _cuda(c)
    mass, mtol = oracle.prompt(c, last)
    _prompt(g, last)
    _within(g["mass"], mass, mtol, "the prompt's mass")
    c["mass"] = g["mass"].cpu()                              # selections are made on the same bits
    k, v, m, kept, length = oracle.evict(c, keep, recent, 400, dst)
    got, n = ops.kv_evict(g["k"], g["v"], g["table"], g["ctx"], g["mass"], keep=keep, recent=recent, max_ctx=400, dst_table=dst.cuda())
    assert torch.equal(got.cpu(), kept) and torch.equal(n.cpu(), length) and _same(g["k"], k) and _same(g["v"], v) and _same(g["mass"], m)
    c.update(k=k, v=v, mass=m, table=dst)
    g.update(table=dst.cuda())
    gen = torch.Generator().manual_seed(61)
    for step in range(20):
        at = n.cpu().long()
        slots = dst[torch.arange(S), at // bs].long() * bs + at % bs
        for name in ("k", "v"):
            row = torch.randn(S, H, D, generator=gen)
            row = (row * 16).to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else row.bfloat16()
            c[name].flatten(0, 1)[slots] = row
            g[name].flatten(0, 1)[slots.cuda()] = row.cuda()
        n = n + 1
        c.update(ctx=n.cpu(), q=torch.randn(S, H * G, D, generator=gen).bfloat16(), q_len=torch.ones(S, dtype=torch.int32), q_start=torch.arange(S, dtype=torch.int32))
        g.update(ctx=n, q=c["q"].cuda())
        c["mass"] = g["mass"].cpu()
        want, tol, mass, mtol = oracle.decode(c)
        _within(_decode(g, max_ctx=keep + 24), want, tol, f"outputs of step {step}")
        _within(g["mass"], mass, mtol, f"mass of step {step}")
    c["mass"] = g["mass"].cpu()
    k, v, m, kept, length = oracle.evict(c, keep, recent, keep + 24)
    got, n = ops.kv_evict(g["k"], g["v"], g["table"], g["ctx"], g["mass"], keep=keep, recent=recent, max_ctx=keep + 24)
    assert torch.equal(got.cpu(), kept) and torch.equal(n.cpu(), length) and _same(g["k"], k) and _same(g["v"], v) and _same(g["mass"], m)


# ----------------------------------------------------------------------------- keys that are no numbers
def _defined(c, last):
    """(mass, outputs of each sequence's last token) of the definition in 64 bits, NaN where a row's softmax has no numbers, and the mass's bound, from what is
    finite of the case: oracle.weights divides rows by their sums whole, so that what such a row does not see would be NaN as well."""
    S, H, D = len(c["ctx"]), c["k"].shape[2], c["k"].shape[3]
    G = c["q"].shape[1] // H
    calm = {**c, **{n: c[n] if c[n].dtype == torch.uint8 else c[n].nan_to_num(0.0, 0.0, 0.0) for n in ("q", "k")}}
    if c["k"].dtype == torch.uint8:
        calm["k"] = torch.where(c["k"] & 0x7f == 0x7f, 0, c["k"])
    mass, tol, out = c["mass"].double().clone(), torch.zeros(c["mass"].shape, dtype=torch.float64), torch.zeros(S, G * H, D, dtype=torch.float64)
    for s in range(S):
        n, ql = int(c["ctx"][s]), int(c["q_len"][s])
        w = min(last or ql, ql)
        if n <= 0 or w <= 0:
            continue
        k = oracle.rows_of(c["k"], c["table"], s, torch.arange(n), c["k_scale"])
        v = oracle.rows_of(c["v"], c["table"], s, torch.arange(n), c["v_scale"])
        q0 = int(c["q_start"][s]) + ql
        for h in range(H):
            z = torch.einsum("wgd,nd->wgn", c["q"][q0 - w:q0, h * G:(h + 1) * G].double(), k[:, h]) * c["scale"]
            seen = (torch.arange(n) < (n - w + 1 + torch.arange(w))[:, None])[:, None].expand_as(z)
            p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            p = torch.where(seen, p, 0.0)
            out[s, h * G:(h + 1) * G] = p[-1] @ v[:, h]
            r = oracle.weight_error(c, D, oracle.weights(calm, s, h, G, last)[1])
            add = p.sum((0, 1))
            mass[s, h, :n] += add
            tol[s, h, :n] = ((r + w * G * 2.0 ** -24) * add + 2.0 ** -23 * mass[s, h, :n]).nan_to_num(0.0) + 1e-30
    return mass, out, tol


def _as_defined(got, want, tol):
    assert torch.equal(got.cpu().isnan(), want.isnan())
    _within(got.cpu().nan_to_num(0.0), want.nan_to_num(0.0), tol, "mass")


def _set_key(c, s, j, h, value, dim=None):
    """Key j of sequence s and kv head h, or one element of it."""
    bs = c["k"].shape[1]
    row = c["k"][int(c["table"][s, j // bs]), j % bs, h]
    if c["k"].dtype == torch.uint8:
        assert math.isnan(value)
        value = 0x7f
    if dim is None:
        row[:] = value
    else:
        row[dim] = value


# what the newest key is alone in: half of a tile, a part of a row's keys, a decode partition (of 512 and of 1024 tokens)
ALONE = [17, 33, 65, 129, 513, 1025, 2049, 4097, 8193]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", ALONE)
@pytest.mark.parametrize("back", [0, 1, 9])
@pytest.mark.parametrize("heads,kv_heads,dim,rows", [(4, 2, 128, 1), (6, 2, 64, 3), (4, 2, 256, 1), (4, 2, 128, 140)])
def test_prompt_of_a_key_that_is_not_a_number(heads, kv_heads, dim, rows, back, n, fp8):
    """Rows that see it have no weights that are numbers, however their keys are cut into parts."""
    c = oracle.case(70, [n, 40], heads, kv_heads, dim, fp8, new=[min(rows, n), 5])
    _set_key(c, 0, n - 1 - back, 0, math.nan, dim // 2)
    want, _, tol = _defined(c, 0)
    g = _cuda(c)
    _prompt(g, 0)
    _as_defined(g["mass"], want, tol)
    assert want[0, 0].isnan().any() and not want[0, 1].isnan().any()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", ALONE)
@pytest.mark.parametrize("back", [0, 1, 700])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (8, 8, 128), (20, 2, 64), (4, 2, 256), (34, 1, 128)])
def test_decode_of_a_key_that_is_not_a_number(heads, kv_heads, dim, back, n, fp8):
    """Its group's outputs and mass are NaN, both of them and whole, however the keys are cut into partitions."""
    c = oracle.case(71, [n, 40], heads, kv_heads, dim, fp8)
    _set_key(c, 0, max(0, n - 1 - back), 0, math.nan, 5)
    want, out, tol = _defined(c, 0)
    g = _cuda(c)
    got = _decode(g)
    _as_defined(g["mass"], want, tol)
    assert torch.equal(got.cpu().isnan(), out.isnan()) and out[0, :heads // kv_heads].isnan().all() and not out[1].isnan().any()


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("n,at", [(65, 64), (1025, 1024), (1025, 3), (4097, 4096), (700, 350)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 4, 128), (8, 2, 128), (3, 3, 256)])
def test_an_infinite_key(heads, kv_heads, dim, n, at, value):
    """A score of -inf is a weight of zero, one of +inf leaves its row no number; heads meet both."""
    c = oracle.case(72, [n, 40], heads, kv_heads, dim, False, new=[1, 1])
    for h in range(kv_heads):
        _set_key(c, 0, at, h, value, 7 + h)
    want, out, tol = _defined(c, 0)
    g = _cuda(c)
    got = _decode(g)
    _as_defined(g["mass"], want, tol)
    assert torch.equal(got.cpu().isnan(), out.isnan())
    g = _cuda(c)
    _prompt(g, 0)
    _as_defined(g["mass"], want, tol)


# ----------------------------------------------------------------------------- queries beyond the range of f16
@pytest.mark.parametrize("apart", [2.0 ** -30, 2.0 ** -9, 2.0 ** 9, 2.0 ** 15, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (12, 1, 64), (20, 1, 128), (30, 1, 128), (33, 1, 128), (16, 2, 256), (8, 8, 64)])
def test_decode_of_rows_far_apart(heads, kv_heads, dim, apart):
    """An e4m3 cache's queries become f16, each row behind a power of two of its own: none loses its range, whatever the rows beside it are. That takes a row's
    largest element to 2^14 at least, where f16 is off by 2^-11 of an element down to 2^-28 of it and by 2^-39 of it below: exact for bf16's eight bits in the
    first case, and in the second less than what the bound has for the products' sum."""
    c = oracle.case(80, [300, 150, 1], heads, kv_heads, dim, True)
    c["scale"] /= max(1.0, apart)
    c["q"][:, ::3] *= apart
    c["q"][1, 5::7] = 0
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    got = _decode(g)
    _within(got, want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


def test_decode_of_the_largest_and_smallest_queries():
    """Elements at either end of bf16 within one row, and rows of subnormal numbers."""
    c = oracle.case(81, [200, 90], 8, 2, 128, True)
    top, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    c["scale"] = 2.0 ** -120
    c["q"][0, 0, ::2], c["q"][0, 1] = top, tiny
    c["q"][0, 2] = torch.where(torch.arange(128) == 5, top, c["q"][0, 2].float()).bfloat16()
    want, tol, mass, mtol = oracle.decode(c)
    g = _cuda(c)
    _within(_decode(g), want, tol, "outputs")
    _within(g["mass"], mass, mtol, "mass")


# ----------------------------------------------------------------------------- more sequences than a launch takes
@pytest.mark.parametrize("own_blocks", [False, True])
def test_evict_of_more_sequences_than_a_launch_takes(own_blocks):
    """One block each, of three rows, the heavier two of which stay: against indexing."""
    S, H, D, bs = 65_540, 1, 64, 4
    g = torch.Generator(device="cuda").manual_seed(90)
    k, v = (torch.randint(0, 256, (2 * S if own_blocks else S, bs, H, D), generator=g, device="cuda", dtype=torch.uint8) for _ in "kv")
    table = torch.randperm(S, generator=g, device="cuda").int().view(S, 1)
    dst = (torch.randperm(S, generator=g, device="cuda").int() + S).view(S, 1) if own_blocks else None
    ctx = torch.full((S,), 3, dtype=torch.int32, device="cuda")
    ctx[::7] = 1
    mass = torch.randperm(4 * S, generator=g, device="cuda").float().view(S, H, 4)          # no two alike
    first, k0, v0 = mass.clone(), k.clone(), v.clone()
    least = first[:, 0, :3].argmin(-1)
    want = torch.stack([(least == 0).long(), 2 - (least == 2).long()], 1)
    want[::7] = torch.tensor([0, -1], device="cuda")
    kept, length = ops.kv_evict(k, v, table, ctx, mass, keep=2, recent=0, max_ctx=3, dst_table=dst)
    assert torch.equal(kept[:, 0].long(), want) and torch.equal(length, ctx.clamp(max=2))
    live, to = want >= 0, (table if dst is None else dst).long()[:, 0]
    assert torch.equal(mass[:, 0, :2], torch.where(live, first[:, 0].gather(1, want.clamp(min=0)), 0.0)) and not mass[:, 0, 2].any() and torch.equal(mass[:, :, 3], first[:, :, 3])
    for new, old in ((k, k0), (v, v0)):
        rows = old[table.long()[:, 0]][torch.arange(S, device="cuda")[:, None], want.clamp(min=0)]
        assert torch.equal(new[to][:, :2][live], rows[live])


def test_prompts_and_decode_of_more_sequences_than_a_launch_takes():
    """Single tokens that see one or two rows: against the weights of two."""
    S, D = 65_540, 64
    g = torch.Generator(device="cuda").manual_seed(91)
    k = torch.randn(S, 2, 1, D, generator=g, device="cuda").bfloat16()
    q = torch.randn(S, 1, D, generator=g, device="cuda").bfloat16()
    ctx = torch.ones(S, dtype=torch.int32, device="cuda")
    ctx[1::3] = 2
    table, start = torch.randperm(S, generator=g, device="cuda").int().view(S, 1), torch.arange(S, dtype=torch.int32, device="cuda")
    z = torch.einsum("sd,snd->sn", q[:, 0].double(), k[table[:, 0].long()][:, :, 0].double()) * D ** -0.5
    z[ctx == 1, 1] = -math.inf
    want = torch.softmax(z, -1)
    for form in ("prompt", "decode"):
        mass = torch.zeros(S, 1, 2, device="cuda")
        if form == "prompt":
            ops.prompt_mass(q, k, table, start, torch.ones_like(start), ctx, mass, max_q_len=1, max_ctx=2, scale=D ** -0.5)
        else:
            ops.paged_attention_mass(q, k, k, table, ctx, mass, max_ctx=2, scale=D ** -0.5)
        # scores of some 50 terms of size one, 64 additions off by 2^-23 of 12 each at most
        assert float((mass[:, 0].double() - want).abs().max()) <= 64 * 2.0 ** -23 * 12


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_whose_scores_are_all_minus_infinity_give_nothing(dim):
    c = oracle.case(74, [1, 700, 1100], 2, 2, dim, False, new=[1, 3, 1])
    c["q"][:, 1, 5] = 1.0
    for s, n in ((0, 1), (1, 699), (2, 1100)):               # all that the only row sees; all but what the newest row sees last; all
        for j in range(n):
            _set_key(c, s, j, 1, -math.inf, 5)
    g = _cuda(c)
    before = g["mass"].clone()
    _prompt(g, 0)
    gained = (g["mass"] - before).double().sum(-1)
    # two of the second sequence's three rows see only what weighs nothing
    assert torch.allclose(gained.cpu(), torch.tensor([[1.0, 0.0], [3.0, 1.0], [1.0, 0.0]]).double(), atol=1e-3)
    before = g["mass"].clone()
    out = _decode({**g, "q": g["q"][[0, 3, 4]].contiguous()})
    assert not out[0, 1].any() and not out[2, 1].any() and not out.isnan().any() and out[1, 1].any()
    gained = (g["mass"] - before).double().sum(-1)
    assert torch.allclose(gained.cpu(), torch.tensor([[1.0, 0.0], [1.0, 1.0], [1.0, 0.0]]).double(), atol=1e-3)


def test_prompt_lanes_without_rows_may_begin_anywhere():
    """Lanes that pad a batch: no rows, so their start is not looked at (the fixture sees that nothing is reported)."""
    c = _cuda(oracle.case(75, [200, 60, 90], 8, 2, 128, False, new=[40, 0, 90]))
    m = c["mass"].clone()
    _prompt(c, 0)
    for start in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        again = m.clone()
        _prompt({**c, "mass": again, "q_start": torch.tensor([0, start, 40], dtype=torch.int32, device="cuda")}, 0)
        ops.check_status("cuda")
        assert _same(again, c["mass"])


# ----------------------------------------------------------------------------- few observers over long contexts, and very many rows
# More parts of a row than a CTA joins by itself (8193 tokens on), parts that grow with the context (16385 on), at one and two tiles of rows
LONG = [8193, 16385, 33000]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", LONG)
@pytest.mark.parametrize("heads,kv_heads,dim,last", [(10, 2, 128, 24), (10, 2, 128, 32), (3, 1, 64, 64), (16, 1, 256, 8), (16, 1, 256, 32), (4, 4, 128, 300)])
def test_prompt_of_a_long_context(heads, kv_heads, dim, last, n, fp8):
    """In a batch with short ones, against 64 bits, and alone with the same bits."""
    ctx, new = [n, 700, 40], [min(n, last + 7), 300, 40]
    c = oracle.case(76, ctx, heads, kv_heads, dim, fp8, new=new)
    mass, mtol = oracle.prompt(c, last)
    g = _cuda(c)
    m = g["mass"].clone()
    _prompt(g, last)
    _within(g["mass"], mass, mtol, "mass")
    for s in range(3):
        one = {k: g[k][s:s + 1] for k in ("table", "ctx", "q_start", "q_len")}
        _prompt({**g, **one, "mass": m[s:s + 1]}, last, max_q_len=new[s], max_ctx=ctx[s])
        assert _same(m[s], g["mass"][s])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("last", [32, 60])
def test_prompt_of_a_long_context_with_keys_that_are_no_numbers(last, fp8):
    """As the first, a middle and the newest key, through the join of many parts."""
    for at in (0, 9000, 16999):
        c = oracle.case(77, [17000, 300], 8, 2, 128, fp8, new=[64, 64])
        _set_key(c, 0, at, 1, math.nan, 3)
        want, _, tol = _defined(c, last)
        g = _cuda(c)
        _prompt(g, last)
        _as_defined(g["mass"], want, tol)


@pytest.mark.parametrize("fp8", [False, True])
def test_prompt_of_more_than_65536_rows(fp8):
    """Where parts of a column are longer than the least: 64 heads a kv head, against 64 bits on the device."""
    n, G, D = 1100, 64, 64
    c = _cuda(oracle.case(78, [n, 50], G, 1, D, fp8, new=[n, 50]))
    before = c["mass"].clone()
    _prompt(c, 0)
    q0 = 0
    for s, m in enumerate((n, 50)):
        k = oracle.rows_of(c["k"], c["table"], s, torch.arange(m, device="cuda"), c["k_scale"])[:, 0]
        add, size = torch.zeros(m, dtype=torch.float64, device="cuda"), 0.0
        unseen = torch.arange(m, device="cuda") > torch.arange(m, device="cuda")[:, None]
        for h in range(G):
            q = c["q"][q0:q0 + m, h].double()
            add += torch.softmax((q @ k.T * c["scale"]).masked_fill(unseen, -math.inf), -1).sum(0)
            size = max(size, float((q.abs() @ k.abs().T).max()) * c["scale"] * oracle.LOG2E)
        q0 += m
        want = before[s, 0, :m].double() + add
        tol = (oracle.weight_error({**c, "k": c["k"].cpu()}, D, size) + m * G * 2.0 ** -24) * add + 2.0 ** -23 * want
        _within(c["mass"][s, 0, :m], want.cpu(), tol.cpu(), f"mass of sequence {s}")


# ----------------------------------------------------------------------------- without programmatic dependence, and with it everywhere
@pytest.mark.parametrize("fp8", [False, True])
def test_the_same_bits_however_kernels_are_launched(fp8):
    """Launches that wait for the one in front as a whole, the default, and all of them programmatic, where each kernel has to wait by itself: a prompt, its
    cut, decode and a cut in place, one behind the other."""
    base = _cuda(oracle.case(79, [900, 130, 2100], 10, 2, 128, fp8, new=[60, 130, 300]))
    gen = torch.Generator(device="cuda").manual_seed(80)
    q1 = torch.randn(3, 10, 128, generator=gen, device="cuda").bfloat16()
    own = (len(base["k"]) + torch.arange(3 * 20, dtype=torch.int32, device="cuda")).view(3, 20)
    spare = torch.zeros(60, *base["k"].shape[1:], dtype=base["k"].dtype, device="cuda")
    lib, results = _native.lib(), []
    default = lib.mb_pdl_enabled()
    try:
        for mode in (0, 1, 2, 1, 0):
            lib.mb_set_pdl(mode)
            c = {**base, "k": torch.cat([base["k"], spare]), "v": torch.cat([base["v"], spare]), "mass": base["mass"].clone()}
            for last in (0, 20):
                _prompt(c, last)
            kept, n = ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=310, recent=10, max_ctx=c["max_ctx"], dst_table=own)
            outs = [_decode({**c, "q": q1, "table": own, "ctx": n}, max_ctx=320) for _ in range(3)]
            again, n2 = ops.kv_evict(c["k"], c["v"], own, n, c["mass"], keep=128, recent=10, max_ctx=320)
            results.append((*outs, kept, n, again, n2, c["mass"], c["k"], c["v"]))
    finally:
        lib.mb_set_pdl(default)
    for r in results[1:]:
        assert all(_same(a, b) for a, b in zip(results[0], r))


@pytest.mark.parametrize("last", [4, 0])
@pytest.mark.parametrize("value", [math.nan, -0.0625])
def test_prompt_of_a_scale_that_is_none(value, last):
    """Scales of a cache are positive: weights behind another are no numbers, and not those of equal scores. A scale of zero makes scores equal."""
    c = _cuda(oracle.case(82, [300, 40], 8, 2, 128, True, new=[300, 3]))
    m = c["mass"].clone()
    _prompt({**c, "k_scale": torch.tensor([value], device="cuda")}, last)
    assert c["mass"][0, :, :300].isnan().all() and c["mass"][1, :, :40].isnan().all()
    c["mass"] = m.clone()
    _prompt({**c, "k_scale": torch.zeros(1, device="cuda")}, 1)
    gained = (c["mass"] - m)[0, :, :300]
    assert torch.allclose(gained, torch.full_like(gained, 4 / 300), rtol=1e-4)
