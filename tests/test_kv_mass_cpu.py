"""The CPU form of the operators that hold a cache to a budget by attention weight, and what they refuse."""
import math
import re
import struct
from pathlib import Path

import pytest
import torch

import kv_mass_oracle as oracle
from metrale_inference_alpha_b200 import ops


def _decode(c, **kw):
    return ops.paged_attention_mass(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["mass"], max_ctx=c["max_ctx"], scale=c["scale"], k_scale=c["k_scale"],
                                    v_scale=c["v_scale"], **kw)


def _prompt(c, last, **kw):
    return ops.prompt_mass(c["q"], c["k"], c["table"], c["q_start"], c["q_len"], c["ctx"], c["mass"], max_q_len=int(c["q_len"].max()), max_ctx=c["max_ctx"],
                           scale=c["scale"], last=last, k_scale=c["k_scale"], **kw)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (5, 1, 128), (3, 3, 256)])
def test_decode_gives_outputs_and_adds_weights(fp8, heads, kv_heads, dim):
    c = oracle.case(1, [33, 0, 1, 17], heads, kv_heads, dim, fp8, columns=40)
    before = c["mass"].clone()
    want, tol, mass, mtol = oracle.decode(c)
    got = _decode(c)
    assert ((got.double() - want).abs() <= tol).all() and ((c["mass"].double() - mass).abs() <= mtol).all()
    assert torch.equal(got[1], torch.zeros_like(got[1])) and torch.equal(c["mass"][1], before[1])
    gained = (c["mass"] - before).double().sum(2)
    assert torch.allclose(gained[0], torch.full_like(gained[0], heads / kv_heads), rtol=1e-4)


@pytest.mark.parametrize("last", [0, 1, 4])
def test_prompt_adds_the_weights_of_its_last_tokens(last):
    c = oracle.case(2, [40, 9, 5, 0], 6, 2, 64, False, new=[7, 9, 1, 0])
    mass, mtol = oracle.prompt(c, last)
    assert _prompt(c, last) is c["mass"]
    assert ((c["mass"].double() - mass).abs() <= mtol).all()


def test_prompt_rows_that_see_nothing_give_nothing():
    c = oracle.case(3, [3], 2, 1, 64, False, new=[5])                     # two of five tokens lie before what is cached
    before = c["mass"].clone()
    _prompt(c, 0)
    assert float((c["mass"] - before).sum()) == pytest.approx(3 * 2, rel=1e-5)


def _poisoned(c, seed):
    g = torch.Generator().manual_seed(seed)
    m = c["mass"]
    m.copy_(torch.randint(0, 6, m.shape, generator=g).float())            # many ties
    for value in (math.nan, math.inf, -math.inf, -0.0):
        m[torch.rand(m.shape, generator=g) < 0.05] = value


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (8, 3), (16, 16), (20, 0), (64, 5)])
@pytest.mark.parametrize("own_blocks", [False, True])
def test_evict_keeps_the_heaviest_and_the_latest(keep, recent, own_blocks):
    c = oracle.case(4, [40, 1, 16, 17, 0], 4, 2, 64, False)
    _poisoned(c, 5)
    nb, dst = c["k"].shape[0], None
    if own_blocks:
        per = (keep + 15) // 16
        dst = (torch.arange(5 * per, dtype=torch.int32) + nb).flip(0).view(5, per)
        c["k"], c["v"] = (torch.cat([x, torch.zeros(5 * per, *x.shape[1:], dtype=x.dtype)]) for x in (c["k"], c["v"]))
    k, v, mass, kept, length = oracle.evict(c, keep, recent, c["max_ctx"], dst)
    got = ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=keep, recent=recent, max_ctx=c["max_ctx"], dst_table=dst)
    assert torch.equal(got[0], kept) and torch.equal(got[1], length)
    for a, b in ((c["k"], k), (c["v"], v), (c["mass"], mass)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_evict_leaves_the_source_mass_where_another_takes_it():
    c = oracle.case(6, [30, 12], 2, 2, 64, True)
    before, out = c["mass"].clone(), torch.full((2, 2, 35), 9.0)
    mass = oracle.evict(c, 10, 2, 30)[2]
    ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=10, recent=2, max_ctx=30, mass_out=out)
    assert torch.equal(c["mass"], before) and torch.equal(out[:, :, :30], mass) and bool((out[:, :, 30:] == 9).all())


# ----------------------------------------------------------------------------- refusals
def _bad_decode():
    yield "q type", dict(q=lambda q: q.float())
    yield "q shape", dict(q=lambda q: q[:1])
    yield "q order", dict(q=lambda q: q.transpose(0, 1).contiguous().transpose(0, 1))
    yield "groups", dict(q=lambda q: q[:, :3].contiguous())
    yield "cache type", dict(k=lambda k: k.float())
    yield "cache order", dict(k=lambda k: k.transpose(1, 2).contiguous().transpose(1, 2))
    yield "v shape", dict(v=lambda v: v[:1])
    yield "head dim", dict(q=lambda q: q[:, :, :32].contiguous(), k=lambda k: k[..., :32].contiguous(), v=lambda v: v[..., :32].contiguous())
    yield "table type", dict(table=lambda t: t.long())
    yield "table rows", dict(table=lambda t: t[:1])
    yield "table width", dict(table=lambda t: t[:, :1])
    yield "lengths type", dict(ctx=lambda x: x.long())
    yield "lengths order", dict(ctx=lambda x: x.repeat_interleave(2)[::2])
    yield "mass type", dict(mass=lambda m: m.double())
    yield "mass columns", dict(mass=lambda m: m[:, :, :20])
    yield "mass order", dict(mass=lambda m: m.transpose(1, 2).contiguous().transpose(1, 2))
    yield "mass shared", dict(mass=lambda m: m[:1].expand(2, -1, -1))
    yield "mass heads", dict(mass=lambda m: m[:, :1])
    yield "scale", dict(scale=lambda x: 0.0)
    yield "negative length", dict(max_ctx=lambda n: -1)


@pytest.mark.parametrize("change", [c for _, c in _bad_decode()], ids=[n for n, _ in _bad_decode()])
def test_decode_refuses(change):
    c = oracle.case(7, [40, 33], 4, 2, 64, False)
    for key, f in change.items():
        c[key] = f(c[key])
    before = c["mass"].clone()
    with pytest.raises(ValueError, match="paged_attention_mass"):
        _decode(c)
    assert torch.equal(c["mass"], before)


def test_decode_refuses_odd_blocks_of_64_byte_rows():
    """A copy into shared memory begins on 128 bytes."""
    for block in (1, 3, 15):
        with pytest.raises(ValueError, match="even number"):
            _decode(oracle.case(12, [40], 4, 2, 64, True, block=block))
        _decode(oracle.case(12, [40], 4, 2, 64, False, block=block))


def test_e4m3_caches_want_scales():
    c = oracle.case(8, [40], 4, 2, 64, True)
    for name in ("k_scale", "v_scale"):
        with pytest.raises(ValueError, match="scales"):
            _decode({**c, name: None})
    with pytest.raises(ValueError, match="scales"):
        _prompt({**c, "k_scale": None}, 1)
    with pytest.raises(ValueError, match="scales"):
        _prompt({**c, "k_scale": c["k_scale"].double()}, 1)


@pytest.mark.parametrize("change", [dict(last=-1), dict(max_q_len=-1), dict(q_start=torch.zeros(2, dtype=torch.int64)), dict(q_len=torch.ones(3, dtype=torch.int32)),
                                    dict(max_ctx=49)], ids=lambda c: next(iter(c)))
def test_prompt_refuses(change):
    c = oracle.case(9, [40, 33], 4, 2, 64, False, new=[5, 6])
    kw = dict(q_start=c["q_start"], q_len=c["q_len"], max_q_len=6, max_ctx=40, last=0) | change
    with pytest.raises(ValueError, match="prompt_mass"):
        ops.prompt_mass(c["q"], c["k"], c["table"], kw.pop("q_start"), kw.pop("q_len"), c["ctx"], c["mass"], scale=c["scale"], **kw)


@pytest.mark.parametrize("change", [dict(keep=0), dict(recent=-1), dict(recent=9), dict(max_ctx=49), dict(mass_out="narrow"), dict(mass_out="overlap"), dict(mass_out="shared"),
                                    dict(dst_table="narrow"), dict(dst_table="type"), dict(dst_table="rows")], ids=lambda c: "-".join(map(str, next(iter(c.items())))))
def test_evict_refuses(change):
    c = oracle.case(10, [40, 33], 4, 2, 64, False)
    big = torch.zeros(2, 2, 60)
    special = {"narrow": dict(mass_out=torch.zeros(2, 2, 39), dst_table=torch.zeros(2, 0, dtype=torch.int32)), "overlap": dict(mass_out=big[:, :, 10:50]),
               "shared": dict(mass_out=torch.zeros(1, 2, 40).expand(2, -1, -1)), "type": dict(dst_table=torch.zeros(2, 1)), "rows": dict(dst_table=torch.zeros(1, 1, dtype=torch.int32))}
    kw = dict(keep=8, recent=2, max_ctx=40)
    for key, v in change.items():
        kw[key] = special[v][key] if isinstance(v, str) else v
    mass = big[:, :, :40] if change.get("mass_out") == "overlap" else c["mass"]
    k = c["k"].clone()
    with pytest.raises(ValueError, match="kv_evict"):
        ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], mass, **kw)
    assert torch.equal(c["k"].nan_to_num(7.0), k.nan_to_num(7.0))


def test_evict_refuses_keys_and_values_that_share_memory():
    """They move side by side: the one would write rows that the other has not read."""
    c = oracle.case(13, [40, 33], 4, 2, 64, False)
    k = c["k"].nan_to_num(0.0)
    both = torch.cat([k, k])
    for v in (k, both[1:1 + len(k)]):
        source = k if v is k else both[:len(k)]
        before = source.clone()
        with pytest.raises(ValueError, match="kv_evict: k_cache and v_cache share memory"):
            ops.kv_evict(source, v, c["table"], c["ctx"], c["mass"], keep=8, recent=2, max_ctx=40)
        assert torch.equal(source, before)
    ops.kv_evict(both[:len(k)], both[len(k):], c["table"], c["ctx"], c["mass"], keep=8, recent=2, max_ctx=40)      # next to each other is not shared


def test_lengths_below_zero_are_zero():
    c = oracle.case(14, [40, 33], 4, 2, 64, False, new=[1, 1])
    c["ctx"][0] = -3
    before = c["mass"].clone()
    _prompt(c, 1)
    c["q"] = c["q"][:2]
    assert not _decode(c)[0].any() and torch.equal(c["mass"][0], before[0])
    kept, length = ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=8, recent=2, max_ctx=40)
    assert length.tolist() == [0, 8] and length.dtype == torch.int32 and bool((kept[0] == -1).all()) and not c["mass"][0].any()


def test_caches_without_heads_or_rows_and_sizes_beyond_32_bits_are_refused():
    c = oracle.case(15, [40, 33], 4, 2, 64, False, new=[1, 1])
    none = dict(k=c["k"][:, :, :0].contiguous(), v=c["v"][:, :, :0].contiguous(), mass=c["mass"][:, :0])
    with pytest.raises(ValueError, match="paged_attention_mass"):
        _decode({**c, **none, "q": c["q"][:2]})
    with pytest.raises(ValueError, match="prompt_mass"):
        _prompt({**c, **none}, 1)
    with pytest.raises(ValueError, match="paged_attention_mass"):
        _decode({**c, "k": c["k"][:, :0].contiguous(), "v": c["v"][:, :0].contiguous(), "q": c["q"][:2], "max_ctx": 0})
    with pytest.raises(ValueError, match="paged_attention_mass"):
        _decode({**c, "k": c["k"][:0], "v": c["v"][:0], "q": c["q"][:2]})
    with pytest.raises(ValueError, match="prompt_mass"):
        ops.prompt_mass(c["q"], c["k"], c["table"], c["q_start"], c["q_len"], c["ctx"], c["mass"], max_q_len=1 << 31, max_ctx=40, scale=1.0, last=1)
    with pytest.raises(ValueError, match="kv_evict"):
        ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=1 << 31, recent=2, max_ctx=40)


def test_nothing_to_do():
    c = oracle.case(11, [4], 2, 1, 64, False)
    none = dict(table=c["table"][:0], ctx=c["ctx"][:0], mass=c["mass"][:0])
    assert ops.paged_attention_mass(c["q"][:0], c["k"], c["v"], none["table"], none["ctx"], none["mass"], max_ctx=4, scale=1.0).shape == (0, 2, 64)
    kept, length = ops.kv_evict(c["k"], c["v"], none["table"], none["ctx"], none["mass"], keep=2, recent=1, max_ctx=4)
    assert kept.shape == (0, 1, 2) and length.shape == (0,)


# ----------------------------------------------------------------------------- cuts that would read what they write
def _cut(c, table, **kw):
    return ops.kv_evict(c["k"], c["v"], table, c["ctx"], c["mass"], **(dict(keep=8, recent=2, max_ctx=40) | kw))


def test_evict_in_place_refuses_sequences_that_share_blocks():
    """One row of a table for all, or rows that overlap: each sequence would move the others' rows."""
    c = oracle.case(16, [40, 40], 4, 2, 64, False)
    wide = torch.arange(1, 6, dtype=torch.int32)
    k = c["k"].clone()
    for table in (c["table"][:1].expand(2, -1), wide.as_strided((2, 3), (1, 1))):
        with pytest.raises(ValueError, match="kv_evict: sequences share rows of block_table"):
            _cut(c, table)
        assert torch.equal(c["k"].view(torch.int16), k.view(torch.int16))
    assert _cut(c, c["table"][:1].expand(2, -1), keep=40)[1].tolist() == [40, 40]                    # nothing moves
    assert _cut({**c, "ctx": c["ctx"][:1], "mass": c["mass"][:1]}, c["table"][:1].expand(1, -1))[1].tolist() == [8]


def test_evict_refuses_blocks_that_several_sequences_are_to_take():
    c = oracle.case(17, [40, 40], 4, 2, 64, False)
    c["k"], c["v"] = (torch.cat([x, torch.zeros(2, *x.shape[1:], dtype=x.dtype)]) for x in (c["k"], c["v"]))
    own = torch.tensor([[len(c["k"]) - 2], [len(c["k"]) - 1]], dtype=torch.int32)
    with pytest.raises(ValueError, match="kv_evict: sequences share rows of dst_table"):
        _cut(c, c["table"], dst_table=own[:1].expand(2, -1))
    assert _cut(c, c["table"], dst_table=own)[1].tolist() == [8, 8]


def test_evict_refuses_its_own_table_as_the_destination():
    """Cuts in place go without dst_table: rows copied to other blocks are written in any order."""
    c = oracle.case(18, [40, 40], 4, 2, 64, False)
    k = c["k"].clone()
    for dst in (c["table"], c["table"][:, :1], c["table"][:, 1:], c["table"].view(2, -1)):
        with pytest.raises(ValueError, match="kv_evict: dst_table and block_table share memory"):
            _cut(c, c["table"], dst_table=dst)
        assert torch.equal(c["k"].view(torch.int16), k.view(torch.int16))


def test_evict_takes_tables_that_lie_beside_each_other():
    """Halves of one buffer's rows, either of them first, and buffers one behind the other."""
    for order in (0, 1):
        c = oracle.case(19, [40, 33], 4, 2, 64, False)
        n = len(c["k"])
        c["k"], c["v"] = (torch.cat([x, torch.zeros(2, *x.shape[1:], dtype=x.dtype)]) for x in (c["k"], c["v"]))
        own = torch.tensor([[n], [n + 1]], dtype=torch.int32)
        both = torch.cat([own, c["table"]] if order else [c["table"], own], 1)
        table, dst = (both[:, 1:], both[:, :1]) if order else (both[:, :3], both[:, 3:])
        k, v, mass, kept, length = oracle.evict(c, 8, 2, 40, own)
        got = _cut(c, table, dst_table=dst)
        assert torch.equal(got[0], kept) and torch.equal(got[1], length) and torch.equal(c["k"].view(torch.int16), k.view(torch.int16))
    c = oracle.case(19, [40, 33], 4, 2, 64, False)
    flat = torch.cat([c["table"].flatten(), torch.tensor([len(c["k"]) - 2, len(c["k"]) - 1], dtype=torch.int32)])
    _cut(c, flat[:6].view(2, 3), dst_table=flat[6:].view(2, 1), keep=3, recent=1)


# ----------------------------------------------------------------------------- what the kernels report
def _state(c):
    return [x.clone().view(torch.uint8) for x in (c["k"], c["v"], c["mass"])]


def test_lengths_and_blocks_out_of_range_are_refused_on_the_cpu():
    """A CUDA call cuts them and sets the status word; here nothing is written."""
    c = oracle.case(21, [40, 33], 4, 2, 64, False, new=[3, 2], columns=50)
    one = {**c, "q": c["q"][:2]}
    before = _state(c)
    bad = c["table"].clone()
    bad[1, 1] = len(c["k"])
    negative = c["table"].clone()
    negative[0, 2] = -1
    for table in (bad, negative):
        with pytest.raises(ValueError, match="paged_attention_mass: .*block"):
            _decode({**one, "table": table})
        with pytest.raises(ValueError, match="prompt_mass: .*block"):
            _prompt({**c, "table": table}, 0)
        with pytest.raises(ValueError, match="kv_evict: .*block"):
            ops.kv_evict(c["k"], c["v"], table, c["ctx"], c["mass"], keep=8, recent=2, max_ctx=40)
        with pytest.raises(ValueError, match="kv_evict: .*block"):
            ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=40, recent=2, max_ctx=40, dst_table=table.clone() - 1000)
    with pytest.raises(ValueError, match="paged_attention_mass: .*max_ctx"):
        _decode({**one, "max_ctx": 39})
    with pytest.raises(ValueError, match="prompt_mass: .*max_ctx"):
        _prompt({**c, "max_ctx": 39}, 0)
    with pytest.raises(ValueError, match="kv_evict: .*max_ctx"):
        ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=8, recent=2, max_ctx=20)
    call = dict(max_q_len=3, max_ctx=40, scale=c["scale"], last=0)
    with pytest.raises(ValueError, match="prompt_mass: .*max_q_len"):
        ops.prompt_mass(c["q"], c["k"], c["table"], c["q_start"], c["q_len"], c["ctx"], c["mass"], **{**call, "max_q_len": 2})
    for start in ([-5, 3], [0, 4]):
        with pytest.raises(ValueError, match="prompt_mass: .*rows of q"):
            ops.prompt_mass(c["q"], c["k"], c["table"], torch.tensor(start, dtype=torch.int32), c["q_len"], c["ctx"], c["mass"], **call)
    assert all(torch.equal(a, b) for a, b in zip(before, _state(c)))


def test_blocks_that_no_row_lies_in_are_not_looked_at():
    """Columns of a table behind a sequence's last block, and rows of sequences without tokens, may hold anything."""
    c = oracle.case(22, [40, 17, 0], 4, 2, 64, False, new=[3, 2, 0])
    c["table"][1, 2], c["table"][2] = 10 ** 6, -7
    before = c["mass"].clone()
    _prompt(c, 0)
    _decode({**c, "q": c["q"][:3]})
    assert torch.equal(c["mass"][2], before[2]) and bool((c["mass"][1, :, :17] != before[1, :, :17]).any())
    assert ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], c["mass"], keep=8, recent=2, max_ctx=40)[1].tolist() == [8, 8, 0]


def test_rows_whose_scores_are_all_minus_infinity_give_nothing():
    """As rows that see nothing, here and in the kernels: no key has a weight."""
    c = oracle.case(23, [1, 20], 2, 2, 64, False, new=[1, 3])
    c["k"][c["table"][0, 0], 0, 1, 5] = -math.inf
    c["q"][0, 1, 5] = 1.0
    before = c["mass"].clone()
    _prompt(c, 0)
    assert float(c["mass"][0, 0, 0]) == pytest.approx(float(before[0, 0, 0]) + 1) and torch.equal(c["mass"][0, 1], before[0, 1]) and not c["mass"].isnan().any()
    out = _decode({**c, "q": c["q"][[0, 3]].contiguous()})
    assert not out[0, 1].any() and out[0, 0].any() and torch.equal(c["mass"][0, 1], before[0, 1]) and not c["mass"].isnan().any()


# ----------------------------------------------------------------------------- packed arguments
def _fields(name):
    """Codes of the struct module for the fields of a C structure of kv_mass.h, in order."""
    path = Path(ops.__file__).parent / "csrc" / "kv_mass.h"
    body = re.search(r"struct %s \{(.*?)\n\};" % name, path.read_text(), re.S).group(1)
    codes = ""
    for decl in re.sub(r"//[^\n]*", "", body).replace("\n", " ").split(";"):
        if not decl.strip():
            continue
        kind, names = re.match(r"\s*(const void\*|void\*|const int\*|int\*|const float\*|float\*|uint32_t\*|long long|size_t|unsigned|int|float)\s+(.*)", decl).groups()
        codes += ("P" if kind.endswith("*") else {"long long": "q", "size_t": "N", "unsigned": "i", "int": "i", "float": "f"}[kind]) * len(names.split(","))
    return codes


@pytest.mark.parametrize("name", ["MbMassArgs", "MbEvictArgs"])
def test_packed_arguments_are_the_structures_of_the_library(name):
    from metrale_inference_alpha_b200.ops import kv_mass
    packed = kv_mass._MASS_ARGS if name == "MbMassArgs" else kv_mass._EVICT_ARGS
    form = packed.format
    assert form[0] == "@" and "".join(code * int(n or 1) for n, code in re.findall(r"(\d*)([A-Za-z])", form) if code != "x") == _fields(name)
    sizes = re.search(r"static_assert\(sizeof\(%s\) == (\d+)" % name, (Path(ops.__file__).parent / "csrc" / "kv_mass.h").read_text())
    assert int(sizes.group(1)) == packed.size


def test_packed_arguments_of_another_size_are_refused(monkeypatch):
    """The launchers copy a structure whole: the sides have to agree on its size before a call is made."""
    from metrale_inference_alpha_b200.ops import kv_mass
    monkeypatch.setattr(kv_mass, "_lib", None)
    size = kv_mass._library().mb_kv_mass_args
    assert [size(0), size(1), size(2)] == [kv_mass._MASS_ARGS.size, kv_mass._EVICT_ARGS.size, 0]
    monkeypatch.setattr(kv_mass, "_lib", None)
    monkeypatch.setattr(kv_mass, "_EVICT_ARGS", struct.Struct(kv_mass._EVICT_ARGS.format + "q"))
    with pytest.raises(RuntimeError, match="build it again"):
        kv_mass._library()


def test_scales_of_several_elements_are_refused():
    """A cache has one scale for its keys and one for its values; the kernels would take the first of several."""
    c = oracle.case(24, [40], 4, 2, 64, True)
    for name in ("k_scale", "v_scale"):
        for wrong in (c[name].repeat(2), torch.ones(2, 1), torch.ones(0)):
            with pytest.raises(ValueError, match="scales of one element"):
                _decode({**c, name: wrong})
    with pytest.raises(ValueError, match="scales of one element"):
        _prompt({**c, "k_scale": torch.ones(2)}, 1)
    before = c["mass"].clone()
    _decode({**c, "k_scale": c["k_scale"][0], "v_scale": c["v_scale"].view(1, 1)})
    assert bool((c["mass"] != before).any())


@pytest.mark.parametrize("cut", ["columns", "columns turned", "heads", "sequences", "lanes"])
def test_evict_takes_mass_and_mass_out_of_one_buffer(cut):
    """Parts of a buffer that share no element, though they lie between each other."""
    c = oracle.case(25, [40, 33, 0], 4, 2, 64, False)
    S, H, n = c["mass"].shape
    big = torch.full({"heads": (S, 2 * H, n), "sequences": (2 * S, H, n), "lanes": (2 * S, H, n)}.get(cut, (S, H, 2 * n + 1)), 9.0)
    mass, out = {"columns": (big[:, :, :n], big[:, :, n:2 * n]), "columns turned": (big[:, :, n + 1:], big[:, :, :n]), "heads": (big[:, :H], big[:, H:]),
                 "sequences": (big[:S], big[S:]), "lanes": (big[::2], big[1::2])}[cut]
    mass.copy_(c["mass"])
    want = oracle.evict(c, 10, 2, 40)
    kept, length = ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], mass, keep=10, recent=2, max_ctx=40, mass_out=out)
    assert torch.equal(kept, want[3]) and torch.equal(out, want[2]) and torch.equal(mass, c["mass"])
    if cut == "columns":
        assert bool((big[:, :, 2 * n] == 9).all())


@pytest.mark.parametrize("shift", [1, 39, 41, 59, 60 * 2 - 1])
def test_evict_refuses_a_mass_out_that_shares_elements_with_mass(shift):
    c = oracle.case(26, [40, 33], 4, 2, 64, False)
    flat = torch.zeros(600)
    mass, out = flat.as_strided((2, 2, 40), (120, 60, 1)), flat.as_strided((2, 2, 40), (120, 60, 1), shift)
    with pytest.raises(ValueError, match="kv_evict: mass_out overlaps mass"):
        ops.kv_evict(c["k"], c["v"], c["table"], c["ctx"], mass, keep=10, recent=2, max_ctx=40, mass_out=out)


def test_the_loop_of_the_readme_keeps_the_row_of_its_token():
    """Run as it stands, on sequences that its budget holds whole."""
    code = re.search(r"```python\n(ops\.prompt_mass.*?)```", (Path(ops.__file__).parents[2] / "README.md").read_text(), re.S).group(1)
    c = oracle.case(27, [40, 33], 4, 2, 64, False, new=[3, 2], columns=4352)
    nb = len(c["k"])
    own = torch.arange(nb, nb + 2 * 272, dtype=torch.int32).view(2, 272)
    k, v = (torch.cat([x, torch.zeros(2 * 272, *x.shape[1:], dtype=x.dtype)]) for x in (c["k"], c["v"]))
    names = dict(ops=ops, q=c["q"], new_q=c["q"][:2].contiguous(), k_cache=k, v_cache=v, table=c["table"], own=own, q_start=c["q_start"], q_len=c["q_len"], ctx=c["ctx"],
                 mass=c["mass"].zero_(), s=c["scale"])
    exec(code.replace("max_q_len=..., max_ctx=...", "max_q_len=3, max_ctx=40").replace("max_ctx=...", "max_ctx=40"), names)
    assert names["n"].tolist() == [41, 34] and bool((names["kept"][:, :, 33] == 33).all())
    gathered = names["mass"].sum(-1)
    assert torch.allclose(gathered, torch.tensor([[4 * 2.0] * 2, [3 * 2.0] * 2]), rtol=1e-4)
