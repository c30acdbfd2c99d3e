"""The operators that verify drafted tokens (adapters, head norms with rotary
positions, tree attention, token selection) against their plain 64-bit forms.

Every result is a whole number that the fixed-point definition fixes bit for
bit, so every comparison is exact.
"""
import numpy as np
import pytest

import verify_ref as ref

pytestmark = pytest.mark.gpu

rd = pytest.importorskip("rasterdet")

ONE = 1 << 32
I32_MIN, I32_MAX = -(2**31), 2**31 - 1


@pytest.fixture(scope="module")
def ctx():
    c = rd.Context(0)
    yield c
    c.close()


class At:
    """A device buffer from its element `offset` on."""

    def __init__(self, buf, offset):
        self.buf, self.ptr = buf, buf.ptr + 4 * offset


def acts(rng, *shape, std=1.0):
    return np.clip(np.round(rng.normal(size=shape) * std * 65536), I32_MIN, I32_MAX).astype(np.int32)


def edges(rng, *shape):
    return rng.choice(np.array([I32_MIN, I32_MIN + 1, I32_MAX, I32_MAX - 1, 0x7F7F7F7F, 0x7F7F7F80, 1 << 23, -(1 << 23),
                                (1 << 23) - 1, 0, 1, -1], dtype=np.int32), size=shape)


# ---------------------------------------------------------------------------
# Head norms and rotation
# ---------------------------------------------------------------------------
def head_case(ctx, rng, hd, heads, rotary, layout, rows, positions, norm=True, gain=True, in_place=False, pad=0,
              shift=0, scaling=0, factor=ONE, low=0, high=0, original=0, amplitude=65536, base=10000 * ONE, eps=4295,
              make=acts, gain_std=0.2):
    width = sum(heads) * hd
    stride = width + pad
    x = make(rng, rows, stride)
    gains = [65536 + acts(rng, hd, std=gain_std) if gain and i < 2 else None for i in range(len(heads))]
    buf = ctx.to_device(np.concatenate([np.zeros(shift, np.int32), x.reshape(-1)]))
    out = buf if in_place else ctx.to_device(np.full(shift + rows * stride, 7, np.int32))
    table = rd.RopeTable(ctx, rotary, max(rotary, 2), base, layout=layout, scaling=scaling, factor=factor,
                         low_turns=low, high_turns=high, original_positions=original, amplitude=amplitude)
    gb = [None if g is None else ctx.to_device(g) for g in gains]
    sets, at = [], 0
    for i, h in enumerate(heads):
        sets.append(rd.HeadRows(At(buf, shift + at), stride, h, out=At(out, shift + at), out_stride=stride, gain=gb[i],
                                norm=norm, rotate=i < 2))
        at += h * hd
    pos = ctx.to_device(np.asarray(positions, dtype=np.uint32))
    ctx.head_norm_rope(table, pos, rows, hd, eps, sets)
    got = out.numpy().reshape(-1)[shift:].reshape(rows, stride)
    freq = ref.frequencies(base, max(rotary, 2), rotary // 2, scaling, factor, low, high, original)
    exp = x.copy() if in_place else np.full_like(x, 7)
    for r in range(rows):
        c = 0
        for i, h in enumerate(heads):
            for _ in range(h):
                exp[r, c:c + hd] = ref.head_row(x[r, c:c + hd], gains[i], eps, norm, freq, int(positions[r]), layout,
                                                amplitude, i < 2)
                c += hd
    assert np.array_equal(got, exp)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("hd,heads,rotary", [(256, (8, 2, 2), 256), (256, (3, 1), 64), (128, (16, 4, 4), 128),
                                             (64, (5,), 64), (16, (4, 1, 1), 16), (80, (3, 1, 1), 38), (96, (6, 2), 34),
                                             (512, (2, 1), 512), (1024, (1, 1), 1024), (600, (2, 1), 300),
                                             (7, (3, 2), 6), (2, (1, 1), 2), (4, (70, 1), 4), (1, (2,), 0),
                                             (255, (2, 1, 1), 254), (513, (1,), 2)])
def test_head_norm_rope_shapes(ctx, layout, hd, heads, rotary):
    rng = np.random.default_rng(hd * 7 + rotary + layout)
    head_case(ctx, rng, hd, heads, rotary, layout, 3, [0, 1, 70001])


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kw", [
    {"norm": False}, {"gain": False}, {"in_place": True}, {"pad": 12}, {"pad": 3}, {"shift": 1}, {"pad": 4, "shift": 4},
    {"in_place": True, "shift": 2, "pad": 1}, {"make": edges}, {"make": edges, "norm": False}, {"eps": 0},
    {"eps": 2**63 - 1}, {"scaling": 1, "factor": 8 * ONE}, {"amplitude": 79164}, {"amplitude": 1},
    {"amplitude": I32_MAX, "norm": False},
    {"scaling": 2, "factor": 8 * ONE, "low": ONE, "high": 4 * ONE, "original": 8192, "amplitude": 70000},
    {"scaling": 2, "factor": 3 * ONE + 12345, "low": 0, "high": 2**63 - 1, "original": 2**32},
    {"base": 500000 * ONE}, {"base": ONE}, {"base": 7 * ONE // 2}])
def test_head_norm_rope_options(ctx, layout, kw):
    rng = np.random.default_rng(17 + layout)
    head_case(ctx, rng, 64, (3, 2, 1), 48, layout, 4, [0, 5, 1_000_003, 2**32 - 1], **kw)


# rows where a product saturates, or could: large values, results past 2^30 from large gains, scales past 2^21 from
# tiny values, cosines above 2, all of them beside rows where none does
def mixed(rng, rows, width):
    x = acts(rng, rows, width, std=300.0 if rng.integers(2) else 1.0)
    x[::2, : width // 2] = edges(rng, (rows + 1) // 2, width // 2)
    return x


def tiny(rng, rows, width):
    return rng.integers(-2, 3, size=(rows, width)).astype(np.int32)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("hd,heads,rotary", [(256, (6, 2, 2), 256), (256, (13, 1), 96), (96, (5, 1, 1), 96), (48, (9, 2), 24),
                                             (30, (3, 2), 30), (512, (2, 1), 512), (768, (2, 1), 256)])
@pytest.mark.parametrize("kw", [{"make": edges}, {"make": mixed}, {"make": tiny, "eps": 0}, {"gain_std": 9000.0},
                                {"gain_std": 9000.0, "in_place": True}, {"amplitude": 200000}, {"amplitude": 131071},
                                {"amplitude": 131072, "norm": False}, {"make": mixed, "norm": False, "in_place": True}])
def test_head_norm_rope_saturates(ctx, layout, hd, heads, rotary, kw):
    rng = np.random.default_rng(hd + rotary + layout)
    head_case(ctx, rng, hd, heads, rotary, layout, 3, [3, 999, 123456], **kw)


def test_head_norm_rope_equals_the_separate_primitives(ctx):
    rng = np.random.default_rng(5)
    rows, heads, hd = 33, 4, 256
    x, g = acts(rng, rows, heads * hd), 65536 + acts(rng, hd, std=0.1)
    a, b, gb = ctx.to_device(x), ctx.to_device(x), ctx.to_device(g)
    ctx.rms_norm(a, rows * heads, hd, gb, 4295)
    ctx.rope_rotate_pairs(a, rows, heads, hd, hd, hd, 10000 * ONE, 9)
    table = rd.RopeTable(ctx, hd, hd, 10000 * ONE)
    pos = ctx.to_device(np.arange(9, 9 + rows, dtype=np.uint32))
    ctx.head_norm_rope(table, pos, rows, hd, 4295, [rd.HeadRows(b, heads * hd, heads, gain=gb)])
    assert np.array_equal(a.numpy(), b.numpy())


def test_head_norm_rope_of_more_rows_than_a_launch(ctx):
    rng = np.random.default_rng(8)
    rows, hd, some = (1 << 22) + 700, 4, 1009  # (rows and positions repeat)
    x, positions = acts(rng, some, hd), np.arange(some, dtype=np.uint32) * 77
    buf = ctx.to_device(np.resize(x, (rows, hd)))
    table = rd.RopeTable(ctx, hd, hd, 10000 * ONE)
    ctx.head_norm_rope(table, ctx.to_device(np.resize(positions, rows)), rows, hd, 4295, [rd.HeadRows(buf, hd, 1)])
    freq = ref.frequencies(10000 * ONE, hd, hd // 2)
    one = np.stack([ref.head_row(t, None, 4295, True, freq, int(p), 0, 65536, True) for t, p in zip(x, positions)])
    assert np.array_equal(buf.numpy().reshape(rows, hd), np.resize(one, (rows, hd)))


def test_head_norm_rope_without_rotation_or_rows(ctx):
    rng = np.random.default_rng(6)
    x = acts(rng, 5, 3 * 20)
    b = ctx.to_device(x)
    ctx.head_norm_rope(None, None, 5, 20, 0, [rd.HeadRows(b, 60, 3, rotate=False)])
    exp = np.concatenate([ref.head_row(x[r, c:c + 20], None, 0, True, [], 0, 0, 65536, False)
                          for r in range(5) for c in (0, 20, 40)])
    assert np.array_equal(b.numpy().reshape(-1), exp)
    out = ctx.empty((5, 60))
    ctx.head_norm_rope(None, None, 5, 20, 0, [rd.HeadRows(b, 60, 3, out=out, norm=False, rotate=False)])
    assert np.array_equal(b.numpy(), out.numpy())
    ctx.head_norm_rope(None, None, 0, 20, 0, [rd.HeadRows(None, 60, 3)])
    ctx.head_norm_rope(None, None, 5, 20, 0, [rd.HeadRows(None, 0, 0)])


def test_rotation_refusals(ctx):
    x = ctx.empty((1, 8))
    ok = dict(rotary_dim=4, freq_base_dim=4, base=ONE * 10)
    for status, kw in [(2, {"rotary_dim": 3}), (2, {"freq_base_dim": 1}), (2, {"freq_base_dim": 0}), (2, {"base": 0}),
                       (2, {"base": 2**63 - 1}), (1, {"layout": 2}), (1, {"scaling": 3}), (1, {"amplitude": 0}),
                       (1, {"amplitude": -1}), (1, {"rotary_dim": 1026}), (1, {"scaling": 1, "factor": ONE - 1}),
                       (1, {"scaling": 2, "low_turns": 5, "high_turns": 5, "original_positions": 9}),
                       (1, {"scaling": 2, "low_turns": -1, "high_turns": 5, "original_positions": 9}),
                       (1, {"scaling": 2, "low_turns": 0, "high_turns": 5, "original_positions": 0})]:
        with pytest.raises(rd.DetError) as e:
            rd.RopeTable(ctx, **{**ok, **kw})
        assert e.value.status == status, kw
    table, pos = rd.RopeTable(ctx, **ok), ctx.to_device(np.zeros(1, np.uint32))
    rows = rd.HeadRows(x, 8, 2)
    bad = rd.HeadRows(x, 8, 2)
    bad.flags = 8
    for status, args in [(1, (None, pos, 1, 4, 0, [rows])), (1, (table, None, 1, 4, 0, [rows])),
                         (2, (table, pos, 1, 4, -1, [rows])), (2, (table, pos, 1, 0, 0, [rows])),
                         (1, (table, pos, 1, 1025, 0, [rows])), (1, (table, pos, 1, 4, 0, [])),
                         (1, (table, pos, 1, 4, 0, [rows] * 5)), (2, (table, pos, 1, 2, 0, [rows])),
                         (1, (table, pos, 1, 4, 0, [rd.HeadRows(x, 7, 2)])),
                         (1, (table, pos, 1, 4, 0, [rd.HeadRows(None, 8, 2)])),
                         (1, (table, pos, 1, 4, 0, [rd.HeadRows(x, 8, 1, out=x, out_stride=9)])),
                         (1, (table, pos, 1, 4, 0, [bad]))]:
        with pytest.raises(rd.DetError) as e:
            ctx.head_norm_rope(*args)
        assert e.value.status == status, args
    ctx.head_norm_rope(table, pos, 1, 4, 0, [rows])  # (and the context goes on)


# ---------------------------------------------------------------------------
# Tree attention
# ---------------------------------------------------------------------------
def tree_masks(rng, drafts):
    out = []
    for d in drafts:
        if d:
            m, _ = rd.tree_masks([int(rng.integers(-1, i)) if i else -1 for i in range(d)])
            out += m.tolist()
    return np.array(out, dtype=np.uint64)


def tree_case(ctx, rng, cached, drafts, heads, kv_heads, hd, ring=(), starts=None, masks=None, make_q=acts, make_k=acts,
              make_v=acts, q_std=None, pad=0, shift=0):
    kw, total = kv_heads * hd, sum(drafts)
    std = 2.0 / np.sqrt(hd) if q_std is None else q_std
    q = make_q(rng, total, heads * hd + pad, **({"std": std} if make_q is acts else {}))
    k, v = make_k(rng, total, kw + pad), make_v(rng, total, kw + pad)
    masks = tree_masks(rng, drafts) if masks is None else np.asarray(masks, dtype=np.uint64)
    views, logical, keep = [], [], []
    for b, n in enumerate(cached):
        ck, cv = make_k(rng, max(n, 1), kw + pad), make_v(rng, max(n, 1), kw + pad)
        first = int(rng.integers(0, n)) if b in ring and n else 0
        kb, vb = (ctx.to_device(np.concatenate([np.zeros(shift, np.int32), np.roll(t, first, 0).reshape(-1)]))
                  for t in (ck, cv))
        keep += [kb, vb]
        views.append(rd.AttnCache(At(kb, shift), At(vb, shift), kw + pad, n, first=first, wrap=n if b in ring and n else 0))
        logical.append((ck[:n, :kw], cv[:n, :kw]))
    dev = lambda t: ctx.to_device(np.concatenate([np.zeros(shift, np.int32), t.reshape(-1)]))  # noqa: E731
    qb, kb, vb, mb = dev(q), dev(k), dev(v), ctx.to_device(masks)
    sb = None if starts is None else ctx.to_device(np.asarray(starts, dtype=np.uint32))
    out = ctx.to_device(np.full((max(total, 1), heads * hd + pad), 7, np.int32))
    ctx.attention_tree(rd.attn_caches(views), rd.u32_array(drafts), At(qb, shift), heads * hd + pad, At(kb, shift),
                       At(vb, shift), kw + pad, mb, sb, heads, kv_heads, hd, out, heads * hd + pad)
    got = out.numpy()[:total]
    exp = ref.attention_tree(logical, drafts, q[:, :heads * hd], k[:, :kw], v[:, :kw], masks, starts, heads, kv_heads, hd)
    assert np.array_equal(got[:, :heads * hd], exp)
    assert (got[:, heads * hd:] == 7).all()


@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 256), (16, 4, 128), (4, 1, 64), (4, 1, 16), (2, 2, 512), (6, 2, 96),
                                               (12, 3, 80), (3, 1, 1), (5, 5, 7), (7, 1, 33), (24, 1, 32), (2, 1, 130)])
@pytest.mark.parametrize("cached,drafts", [([0], [1]), ([1], [1]), ([63, 0, 64, 65], [1, 3, 2, 4]), ([130], [17])])
def test_tree_attention_shapes(ctx, heads, kv_heads, hd, cached, drafts):
    rng = np.random.default_rng(heads * 1000 + hd + len(cached))
    tree_case(ctx, rng, cached, drafts, heads, kv_heads, hd)


@pytest.mark.parametrize("cached,drafts", [([700], [1]), ([1000, 513, 2], [5, 64, 33]), ([257], [64]), ([40, 50], [0, 9]),
                                           ([31] * 45, [1, 2] * 22 + [3]), ([0] * 3, [64, 1, 0])])
def test_tree_attention_lengths(ctx, cached, drafts):
    rng = np.random.default_rng(sum(cached) + sum(drafts))
    tree_case(ctx, rng, cached, drafts, 4, 1, 64)


@pytest.mark.parametrize("kw", [{"pad": 4}, {"pad": 3}, {"shift": 1}, {"pad": 8, "shift": 4}])
@pytest.mark.parametrize("hd", [64, 30])
def test_tree_attention_strides_and_alignment(ctx, hd, kw):
    tree_case(ctx, np.random.default_rng(hd), [77, 5], [3, 6], 4, 2, hd, ring=(0,), **kw)


def test_tree_attention_rings_and_starts(ctx):
    rng = np.random.default_rng(3)
    cached, drafts = [128, 100, 300, 64], [4, 20, 9, 3]
    starts = rng.integers(0, 140, size=sum(drafts))
    starts[:4] = [127, 128, 129, 2**32 - 1]
    tree_case(ctx, rng, cached, drafts, 8, 2, 64, ring=(0, 1, 2), starts=starts)


def test_tree_attention_rows_that_see_nothing(ctx):
    rng = np.random.default_rng(4)
    # no cache, no bits; no cache, only bits past the drafted rows; everything masked by the start
    masks = [0, 1 << 63 | 1 << 40, 2, 0, 0, 7 << 3]
    tree_case(ctx, rng, [0, 50], [3, 3], 4, 2, 64, masks=masks, starts=[0, 0, 0, 50, 49, 60])
    tree_case(ctx, rng, [0], [1], 4, 1, 16, masks=[0])


def test_tree_attention_sees_later_rows_and_not_itself(ctx):
    rng = np.random.default_rng(5)
    masks = rng.integers(0, 2**63, size=64, dtype=np.uint64) * 2 + rng.integers(0, 2, size=64, dtype=np.uint64)
    tree_case(ctx, rng, [70], [64], 4, 1, 64, masks=masks)


@pytest.mark.parametrize("q,k,v", [(edges, edges, edges), (acts, edges, acts), (edges, acts, acts), (acts, acts, edges)])
@pytest.mark.parametrize("hd", [64, 256, 20])
def test_tree_attention_extremes(ctx, q, k, v, hd):
    tree_case(ctx, np.random.default_rng(hd), [200, 33], [7, 2], 4, 1, hd, make_q=q, make_k=k, make_v=v, ring=(1,))


@pytest.mark.parametrize("n", [3, 100, 1000])
def test_tree_attention_equal_scores(ctx, n):
    # every key alike: the first visible row takes the residual, whatever its sign
    same = lambda rng, r, w: np.tile(acts(np.random.default_rng(1), 1, w), (r, 1))  # noqa: E731
    tree_case(ctx, np.random.default_rng(n), [n], [3], 4, 2, 64, make_k=same, starts=[0, 2, n])


@pytest.mark.parametrize("q_std", [0.0, 0.01, 1.0, 40.0])
def test_tree_attention_spreads(ctx, q_std):
    tree_case(ctx, np.random.default_rng(8), [333], [6], 4, 1, 128, q_std=q_std)


@pytest.mark.parametrize("n", [4097, 20000])
def test_tree_attention_long_cache(ctx, n):
    rng = np.random.default_rng(n)
    tree_case(ctx, rng, [n, 90], [2, 1], 2, 1, 64, starts=[0, n - 300, 5], q_std=0.05)


@pytest.mark.parametrize("q,k,v", [(acts, acts, acts), (acts, edges, acts), (edges, acts, acts), (acts, acts, edges)])
@pytest.mark.parametrize("hd,pad", [(64, 0), (100, 0), (192, 0), (256, 0), (256, 3), (320, 0)])
def test_tree_attention_many_rows(ctx, q, k, v, hd, pad):
    # more than 64 query rows of a head: blocks of 128 rows, whose keys are loaded a step ahead
    tree_case(ctx, np.random.default_rng(hd + pad), [150, 20], [33, 9], 4, 1, hd, make_q=q, make_k=k, make_v=v, ring=(0,),
              pad=pad, starts=np.arange(42) * 3)


@pytest.mark.parametrize("n,drafts", [(4030, 1), (4097, 1), (5000, 64), (16330, 64), (16400, 64)])
def test_tree_attention_whole_rows_and_chunks(ctx, n, drafts):
    # rows turned into weights whole: up to 4096 keys, or 256 rows of up to 16384. The last, first and middle rows
    # against the plain form, all of them against calls of eight rows
    rng = np.random.default_rng(n)
    heads, hd = 4, 16
    k, v = acts(rng, n, hd), acts(rng, n, hd)
    q, dk, dv = acts(rng, drafts, heads * hd, std=0.4), acts(rng, drafts, hd), acts(rng, drafts, hd)
    masks = tree_masks(rng, [drafts])
    starts = rng.integers(0, n, size=drafts).astype(np.uint32)
    starts[::2] = 0
    kb, vb, qb, dkb, dvb = (ctx.to_device(t) for t in (k, v, q, dk, dv))
    mb, sb, out = ctx.to_device(masks), ctx.to_device(starts), ctx.empty((drafts, heads * hd))
    view = rd.attn_caches([rd.AttnCache(kb, vb, hd, n)])
    ctx.attention_tree(view, rd.u32_array([drafts]), qb, heads * hd, dkb, dvb, hd, mb, sb, heads, 1, hd, out, heads * hd)
    got = out.numpy()
    for i in {0, drafts // 2, drafts - 1}:
        seen = [j for j in range(drafts) if int(masks[i]) >> j & 1]
        keys, values = (np.concatenate([c[starts[i]:], d[seen]]) for c, d in ((k, dk), (v, dv)))
        for h in (0, heads - 1):
            c = slice(h * hd, (h + 1) * hd)
            assert np.array_equal(got[i, c], ref.attention_row(q[i, c], keys, values)), (i, h)
    # (two heads of a call at a time: half the rows)
    half = ctx.empty((drafts, 2 * hd))
    for h in (0, 2):
        qh = ctx.to_device(np.ascontiguousarray(q[:, h * hd:(h + 2) * hd]))
        ctx.attention_tree(view, rd.u32_array([drafts]), qh, 2 * hd, dkb, dvb, hd, mb, sb, 2, 1, hd, half, 2 * hd)
        assert np.array_equal(got[:, h * hd:(h + 2) * hd], half.numpy())


def test_tree_attention_scores_past_a_launch(ctx):
    # 512 rows of 70030 keys for each of two kv heads are more score rows than a launch takes: a kv head at a time
    rng = np.random.default_rng(21)
    n, drafts, heads, kv_heads, hd = 69970, 64, 16, 2, 8
    k, v = acts(rng, n, kv_heads * hd), acts(rng, n, kv_heads * hd)
    q, dk, dv = acts(rng, drafts, heads * hd, std=0.5), acts(rng, drafts, kv_heads * hd), acts(rng, drafts, kv_heads * hd)
    masks = tree_masks(rng, [drafts])
    out = ctx.empty((drafts, heads * hd))
    ctx.attention_tree(rd.attn_caches([rd.AttnCache(ctx.to_device(k), ctx.to_device(v), kv_heads * hd, n)]),
                       rd.u32_array([drafts]), ctx.to_device(q), heads * hd, ctx.to_device(dk), ctx.to_device(dv),
                       kv_heads * hd, ctx.to_device(masks), None, heads, kv_heads, hd, out, heads * hd)
    got = out.numpy()
    for i, h in [(0, 0), (63, 7), (30, 8), (63, 15)]:
        seen = [j for j in range(drafts) if int(masks[i]) >> j & 1]
        c, d = slice(h * hd, (h + 1) * hd), slice(h // 8 * hd, (h // 8 + 1) * hd)
        keys, values = np.concatenate([k[:, d], dk[seen][:, d]]), np.concatenate([v[:, d], dv[seen][:, d]])
        assert np.array_equal(got[i, c], ref.attention_row(q[i, c], keys, values)), (i, h)


@pytest.mark.parametrize("cached,drafts,ring,hd,v", [
    ([1500, 700], [20, 17], (0, 1), 256, acts), ([640, 64, 63], [14, 64, 9], (), 256, acts), ([900], [33], (0,), 132, acts),
    ([333, 1], [12, 12], (0,), 512, acts), ([450, 200], [16, 9], (1,), 256, edges)])
def test_tree_attention_long_values(ctx, cached, drafts, ring, hd, v):
    # more than 32 query rows of more than 128 dims: the values come through LDS, over many steps, rings that wrap
    # inside a step and drafted rows at the end of one
    rng = np.random.default_rng(sum(cached) + hd)
    tree_case(ctx, rng, cached, drafts, 4, 1, hd, ring=ring, make_v=v)


def test_tree_attention_far_apart_rows(ctx):
    # rows too far apart for 32-bit offsets of a step, of more than 32 query rows
    rng = np.random.default_rng(13)
    heads, hd, n, stride, d = 16, 160, 70, 1 << 22, 3
    big = ctx.alloc((n - 1) * stride * 4 + 2 * hd * 4)
    k, v = acts(rng, n, hd), acts(rng, n, hd)
    for r in range(n):
        for i, t in enumerate((k, v)):
            row = np.ascontiguousarray(t[r])
            ctx.check(ctx.lib.det_memcpy_h2d(ctx.handle, rd.C.c_void_p(big.ptr + (r * stride + i * hd) * 4),
                                             rd._ptr(row), row.nbytes))
    q, dk, dv = acts(rng, d, heads * hd, std=0.2), acts(rng, d, hd), acts(rng, d, hd)
    masks = np.array([1, 3, 5], dtype=np.uint64)
    out = ctx.empty((d, heads * hd))
    ctx.attention_tree(rd.attn_caches([rd.AttnCache(big, At(big, hd), stride, n)]), rd.u32_array([d]), ctx.to_device(q),
                       heads * hd, ctx.to_device(dk), ctx.to_device(dv), hd, ctx.to_device(masks), None, heads, 1, hd, out,
                       heads * hd)
    assert np.array_equal(out.numpy(), ref.attention_tree([(k, v)], [d], q, dk, dv, masks, None, heads, 1, hd))
    big.free()


def test_tree_attention_offsets_past_32_bits(ctx):
    # rows 4194304 values apart: the last of 1100 lies past 2^32 values (17 GB)
    rng = np.random.default_rng(9)
    hd, n, stride = 64, 1100, 1 << 22
    big = ctx.alloc((n - 1) * stride * 4 + 2 * hd * 4)
    k, v = acts(rng, n, hd), acts(rng, n, hd)
    for r in range(n):
        for i, t in enumerate((k, v)):
            row = np.ascontiguousarray(t[r])
            ctx.check(ctx.lib.det_memcpy_h2d(ctx.handle, rd.C.c_void_p(big.ptr + (r * stride + i * hd) * 4),
                                             rd._ptr(row), row.nbytes))
    q, dk, dv = acts(rng, 2, hd, std=0.3), acts(rng, 2, hd), acts(rng, 2, hd)
    masks = np.array([1, 3], dtype=np.uint64)
    out = ctx.empty((2, hd))
    ctx.attention_tree(rd.attn_caches([rd.AttnCache(big, At(big, hd), stride, n)]), rd.u32_array([2]), ctx.to_device(q),
                       hd, ctx.to_device(dk), ctx.to_device(dv), hd, ctx.to_device(masks), None, 1, 1, hd, out, hd)
    assert np.array_equal(out.numpy(), ref.attention_tree([(k, v)], [2], q, dk, dv, masks, None, 1, 1, hd))
    big.free()


def test_tree_attention_of_a_chain_equals_causal_attention(ctx):
    rng = np.random.default_rng(10)
    heads, kv_heads, hd, n, d = 8, 2, 256, 300, 40
    k, v, q = acts(rng, n + d, kv_heads * hd), acts(rng, n + d, kv_heads * hd), acts(rng, n + d, heads * hd, std=0.2)
    kb, vb, qb = ctx.to_device(k), ctx.to_device(v), ctx.to_device(q)
    causal, out = ctx.empty((n + d, heads * hd)), ctx.empty((d, heads * hd))
    ctx.attention(qb, kb, vb, n + d, n + d, heads, kv_heads, hd, 0, causal)
    masks, _ = rd.tree_masks([-1] + list(range(d - 1)))
    kw = kv_heads * hd
    ctx.attention_tree(rd.attn_caches([rd.AttnCache(kb, vb, kw, n)]), rd.u32_array([d]), At(qb, n * heads * hd),
                       heads * hd, At(kb, n * kw), At(vb, n * kw), kw, ctx.to_device(masks), None, heads, kv_heads, hd,
                       out, heads * hd)
    assert np.array_equal(out.numpy(), causal.numpy()[n:])


def test_tree_attention_refusals(ctx):
    b = ctx.empty((4, 64))
    m = ctx.to_device(np.ones(4, np.uint64))
    good = dict(caches=[rd.AttnCache(b, b, 64, 4)], drafts=[2], q=b, qs=64, k=b, v=b, ks=64, m=m, s=None, nh=4, nkv=4,
                hd=16, out=b, os=64)

    def call(**kw):
        a = {**good, **kw}
        ctx.attention_tree(rd.attn_caches(a["caches"]), rd.u32_array(a["drafts"]), a["q"], a["qs"], a["k"], a["v"],
                           a["ks"], a["m"], a["s"], a["nh"], a["nkv"], a["hd"], a["out"], a["os"])

    for kw in [{"nkv": 0}, {"nh": 3}, {"nh": 6}, {"hd": 0}, {"hd": 513}, {"drafts": [65]}, {"qs": 63}, {"ks": 63},
               {"os": 63}, {"q": None}, {"k": None}, {"v": None}, {"m": None}, {"out": None},
               {"caches": [rd.AttnCache(b, b, 64, (1 << 20) + 1)]}, {"caches": [rd.AttnCache(None, b, 64, 4)]},
               {"caches": [rd.AttnCache(b, None, 64, 4)]}, {"caches": [rd.AttnCache(b, b, 63, 4)]},
               {"caches": [rd.AttnCache(b, b, 64, 4, first=4, wrap=4)]},
               {"caches": [rd.AttnCache(b, b, 64, 4, first=0, wrap=3)]}]:
        with pytest.raises(rd.DetError) as e:
            call(**kw)
        assert e.value.status == 1, kw
    with pytest.raises(ValueError):
        call(drafts=[1, 1])
    out = ctx.empty((4, 64))
    call(out=out)
    call(drafts=[0])
    call(caches=[], drafts=[])


def test_tree_attention_over_layer_caches(ctx):
    # the caches that layer prefills and decodes fill: a full ring and a linear one
    cfg, tensors = fixtures_model()
    model = rd.Model(ctx, cfg)
    for name, val, s in tensors:
        model.set_tensor(name, val, s)
    model.finalize()
    ops = rd.LayerOps(model)
    rng = np.random.default_rng(12)
    n, hidden = 150, 64
    x, y = ctx.to_device(acts(rng, n, hidden)), ctx.empty((n, hidden))
    for layer in range(2):
        cache = rd.KvCache(model, layer, 400)
        with pytest.raises(rd.DetError):
            cache.view()
        ops.layer_prefill(layer, x, n, None, None, cache, y)
        ops.layer_decode(layer, x, None, cache, None, n, y)
        length, kv_heads, hd, _ = cache.info()
        k, v = cache.read_logical()
        rows = [t.transpose(1, 0, 2).reshape(length, kv_heads * hd) for t in (k, v)]
        q, dk, dv = acts(rng, 3, 4 * hd), acts(rng, 3, kv_heads * hd), acts(rng, 3, kv_heads * hd)
        masks = np.array([1, 3, 5], dtype=np.uint64)
        out = ctx.empty((3, 4 * hd))
        ctx.attention_tree(rd.attn_caches([cache.view()]), rd.u32_array([3]), ctx.to_device(q), 4 * hd, ctx.to_device(dk),
                           ctx.to_device(dv), kv_heads * hd, ctx.to_device(masks), None, 4, kv_heads, hd, out, 4 * hd)
        exp = ref.attention_tree([rows], [3], q, dk, dv, masks, None, 4, kv_heads, hd)
        assert np.array_equal(out.numpy(), exp)


def fixtures_model():
    from rasterdet import synthetic

    return synthetic.tiny_model(seed=7)


# ---------------------------------------------------------------------------
# Adapters
# ---------------------------------------------------------------------------
def weights(rng, rows, cols, kind):
    """(values, row scale or None, weight bits)"""
    if kind == "int8":
        q, s = rng.integers(-127, 128, size=(rows, cols), dtype=np.int8), rng.integers(1, 41, size=rows).astype(np.int32)
        return q, s, ref.bits(q, s)
    lim = 32767 if kind == "i16" else 2**31 // (2 * cols + 2)
    w = rng.integers(-lim, lim + 1, size=(rows, cols)).astype(np.int16 if kind == "i16" else np.int32)
    w[:, 0] = 1
    return w, None, w.astype(np.int32)


def adapter_case(ctx, rng, rows, cols, ranks, m, index, kinds=("int8", "int8", "int8"), make=acts, scales=None):
    w = weights(rng, rows, cols, kinds[0])
    ads = [(weights(rng, r, cols, kinds[1]), weights(rng, rows, r, kinds[2]),
            int(rng.integers(-200000, 200000)) if scales is None else scales[i]) for i, r in enumerate(ranks)]
    mat = ctx.upload_matrix(w[0], w[1])
    group = rd.Adapters(ctx, rows, cols, [rd.Adapter(a[0], b[0], s, down_scale=a[1], up_scale=b[1]) for a, b, s in ads])
    x = make(rng, m, cols)
    index = np.asarray(index, dtype=np.uint32)
    out = ctx.to_device(np.full((m + 1, rows), 7, np.int32))
    ctx.det_linear_adapters(mat, group, m, ctx.to_device(x), ctx.to_device(index), out)
    got = out.numpy()
    assert np.array_equal(got[:m], ref.linear_adapters(w[2], [(a[2], b[2], s) for a, b, s in ads], x, index))
    assert (got[m] == 7).all()


@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 64), (33, 130), (130, 33), (257, 1000), (64, 2560)])
@pytest.mark.parametrize("kinds", [("int8", "int8", "int8"), ("i16", "i16", "i16"), ("i32", "i32", "i32"),
                                   ("int8", "i16", "int8"), ("i16", "int8", "i32")])
def test_adapter_shapes_and_types(ctx, rows, cols, kinds):
    rng = np.random.default_rng(rows * 10 + cols)
    ranks = [1, 8, 16, 17]
    m = 19
    adapter_case(ctx, rng, rows, cols, ranks, m, rng.integers(0, 6, size=m), kinds=kinds)


@pytest.mark.parametrize("rank", [1, 15, 16, 31, 64, 65, 128, 200, 256])
def test_adapter_ranks(ctx, rank):
    rng = np.random.default_rng(rank)
    adapter_case(ctx, rng, 70, 200, [rank, 3], 5, [0, 1, 0, 9, 0], kinds=("int8", "int8", "i16"))


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 64, 100])
@pytest.mark.parametrize("mix", ["own", "one", "none", "runs"])
def test_adapter_rows(ctx, m, mix):
    rng = np.random.default_rng(m)
    index = {"own": np.arange(m) % 18, "one": np.full(m, 2), "none": np.full(m, rd.DET_NO_ADAPTER, dtype=np.uint32),
             "runs": np.sort(rng.integers(0, 4, size=m))}[mix]
    adapter_case(ctx, rng, 48, 96, [4, 8, 2, 16] * 4 + [5], m, index)


@pytest.mark.parametrize("kinds", [("int8",) * 3, ("i16",) * 3, ("i32",) * 3])
def test_adapter_extremes(ctx, kinds):
    rng = np.random.default_rng(2)
    adapter_case(ctx, rng, 40, 300, [9, 33], 6, [0, 1, 0, 1, 1, 0], kinds=kinds, make=edges,
                 scales=[I32_MAX, I32_MIN])


@pytest.mark.parametrize("rank", [16, 128, 256])
@pytest.mark.parametrize("value", [-32896, -128, 32639, -(2**23) - 2**15 - 128, 8355711])
def test_adapter_digit_sums_at_their_ends(ctx, rank, value):
    # h and B of one value whose digits are all the lowest or the highest
    ones = np.full((rank, 1), 65536, dtype=np.int32)
    up = np.full((20, rank), value if abs(value) < 2**16 else value // 512, dtype=np.int32)
    x = np.array([[value], [-value]], dtype=np.int32)
    w = np.zeros((20, 1), dtype=np.int32)
    group = rd.Adapters(ctx, 20, 1, [rd.Adapter(ones, up, 65536)])
    out = ctx.empty((2, 20))
    ctx.det_linear_adapters(ctx.upload_matrix(w), group, 2, ctx.to_device(x), ctx.to_device(np.zeros(2, np.uint32)), out)
    assert np.array_equal(out.numpy(), ref.linear_adapters(w, [(ones, up, 65536)], x, [0, 0]))


@pytest.mark.parametrize("rows", [600, 5000, 20011])
def test_adapter_outputs_per_workgroup(ctx, rows):
    # one to four of B's tiles per wave, and rows of every adapter
    rng = np.random.default_rng(rows)
    adapter_case(ctx, rng, rows, 24, [3, 16, 20] * 6, 66, np.arange(66) % 19)


def test_adapter_rows_in_ranges(ctx):
    # more rows than a range of the call, of more adapters than threads that sort them
    rng = np.random.default_rng(7)
    m, rows, cols, n = 8200, 3, 5, 1100
    w = weights(rng, rows, cols, "i16")
    ads = [(weights(rng, 2, cols, "i16"), weights(rng, rows, 2, "i16")) for _ in range(n)]
    index = rng.integers(0, n + 40, size=m).astype(np.uint32)
    x = acts(rng, m, cols)
    group = rd.Adapters(ctx, rows, cols, [rd.Adapter(a[0], b[0], 65536) for a, b in ads])
    out = ctx.empty((m, rows))
    ctx.det_linear_adapters(ctx.upload_matrix(w[0]), group, m, ctx.to_device(x), ctx.to_device(index), out)
    assert np.array_equal(out.numpy(), ref.linear_adapters(w[2], [(a[2], b[2], 65536) for a, b in ads], x, index))


def test_adapter_long_rows(ctx):
    rng = np.random.default_rng(3)
    adapter_case(ctx, rng, 20, 33000, [5], 3, [0, 0, 1])


def test_adapters_equal_the_separate_primitives(ctx):
    rng = np.random.default_rng(4)
    rows, cols, m = 2048, 2560, 40
    w, a, b = weights(rng, rows, cols, "int8"), weights(rng, 24, cols, "i16"), weights(rng, rows, 24, "i16")
    mw, ma, mb = ctx.upload_matrix(w[0], w[1]), ctx.upload_matrix(a[0]), ctx.upload_matrix(b[0])
    x = ctx.to_device(acts(rng, m, cols))
    out, h, d, got = ctx.empty((m, rows)), ctx.empty((m, 24)), ctx.empty((m, rows)), ctx.empty((m, rows))
    ctx.det_linear_slab(mw, m, x, out)
    ctx.det_linear_slab(ma, m, x, h)
    ctx.det_linear_slab(mb, m, h, d)
    ctx.elementwise(rd.DET_EW_SCALE, d, None, m * rows, 50000)
    ctx.elementwise(rd.DET_EW_ADD, out, d, m * rows)
    group = rd.Adapters(ctx, rows, cols, [rd.Adapter(a[0], b[0], 50000)])
    ctx.det_linear_adapters(mw, group, m, x, ctx.to_device(np.zeros(m, np.uint32)), got)
    assert np.array_equal(got.numpy(), out.numpy())


def test_adapter_refusals(ctx):
    rng = np.random.default_rng(6)
    w = weights(rng, 8, 12, "i16")[0]
    mat, small = ctx.upload_matrix(w), ctx.upload_matrix(w[:4].copy())
    down, up = w[:3, :12].copy(), weights(rng, 8, 3, "i16")[0]
    group = rd.Adapters(ctx, 8, 12, [rd.Adapter(down, up)])
    b, idx = ctx.empty((4, 12)), ctx.to_device(np.zeros(4, np.uint32))
    big = np.full((1, 70000), 32767, dtype=np.int16)
    for args in [(8, 12, []), (0, 12, [rd.Adapter(down, up[:0])]), (8, 0, [rd.Adapter(down[:, :0], up)]),
                 (8, 12, [rd.Adapter(np.zeros((257, 12), np.int16), np.zeros((8, 257), np.int16))]),
                 (8, 12, [rd.Adapter(np.zeros((0, 12), np.int16), np.zeros((8, 0), np.int16))]),
                 (1, 70000, [rd.Adapter(big, np.ones((1, 1), np.int16))]),
                 (1, 130001, [rd.Adapter(np.zeros((1, 130001), np.int16), np.ones((1, 1), np.int16))])]:
        with pytest.raises(rd.DetError) as e:
            rd.Adapters(ctx, *args)
        assert e.value.status == 1
    for args in [(small, group, 4, b, idx, b), (mat, group, 4, None, idx, b), (mat, group, 4, b, None, b),
                 (mat, group, 4, b, idx, None)]:
        with pytest.raises(rd.DetError) as e:
            ctx.det_linear_adapters(*args)
        assert e.value.status == 1
    ctx.det_linear_adapters(mat, group, 0, None, None, None)
    other = rd.Context(0)
    with pytest.raises(rd.DetError):
        other.det_linear_adapters(mat, group, 4, b, idx, b)
    other.close()


# ---------------------------------------------------------------------------
# Token selection
# ---------------------------------------------------------------------------
def select_case(ctx, rng, n, vocab, history=20, spans=2, penalties=None, biases=5, masked=True, in_place=False, pad=0,
                make=acts, ids=None, want_out=True, want_tokens=True, mask_pad=0, shift=0):
    x = make(rng, n, vocab + pad)
    if penalties is None:
        penalties = np.stack([rng.integers(30000, 200000, size=n), rng.integers(-5000, 50000, size=n),
                              rng.integers(-5000, 50000, size=n)], 1).astype(np.int32)
    ids = rng.integers(0, vocab + 3, size=history).astype(np.uint32) if ids is None else np.asarray(ids, dtype=np.uint32)
    sp = np.sort(rng.integers(0, len(ids) + 3, size=(n, spans, 2)), axis=-1).astype(np.uint32)
    begin = np.concatenate([[0], np.cumsum(rng.integers(0, 2 * biases + 1, size=n))]).astype(np.uint32)
    bi = rng.integers(0, vocab + 2, size=max(int(begin[-1]), 1)).astype(np.uint32)
    bi[::3] = bi[0]  # (the same token more than once)
    bv = make(rng, bi.size)
    words = (vocab + 31) // 32 + mask_pad
    mask = rng.integers(0, 2**32, size=(n, words), dtype=np.uint64).astype(np.uint32)
    if masked and n > 1:
        mask[1] = 0  # nothing is left
        if vocab % 32:
            mask[1, (vocab - 1) // 32] = np.uint32(0xFFFFFFFF << (vocab % 32) & 0xFFFFFFFF)  # (bits past the vocabulary)
    flat = np.concatenate([np.zeros(shift, np.int32), x.reshape(-1)])
    xb = ctx.to_device(flat)
    ob = xb if in_place else ctx.to_device(np.full(flat.size, 7, np.int32))
    tb = ctx.empty(n, np.uint32)
    rules = rd.LogitRules(penalties=ctx.to_device(penalties), ids=ctx.to_device(ids), n_ids=len(ids),
                          spans=ctx.to_device(sp), spans_per_row=spans, bias_begin=ctx.to_device(begin),
                          bias_ids=ctx.to_device(bi), bias_values=ctx.to_device(bv), n_bias=int(begin[-1]),
                          mask=ctx.to_device(mask) if masked else None, mask_stride=words)
    ctx.select_tokens(At(xb, shift), n, vocab, vocab + pad, rules, At(ob, shift) if want_out else None, vocab + pad,
                      tb if want_tokens else None)
    exp, tok = ref.select(x[:, :vocab], penalties, ids, [[(int(a), int(b)) for a, b in r] for r in sp],
                          [list(zip(bi[b:e].tolist(), bv[b:e].tolist())) for b, e in zip(begin[:-1], begin[1:])],
                          mask if masked else None)
    got = ob.numpy().reshape(-1)[shift:].reshape(n, vocab + pad)
    if want_out:
        assert np.array_equal(got[:, :vocab], exp)
        assert np.array_equal(got[:, vocab:], x[:, vocab:] if in_place else np.full((n, pad), 7))
    if want_tokens:
        assert np.array_equal(tb.numpy(), tok)


@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 2), (2, 31), (2, 32), (2, 33), (5, 512), (2, 4095), (2, 4096), (2, 4097),
                                     (1, 8193), (3, 12345), (1, 50001)])
@pytest.mark.parametrize("masked", [True, False])
def test_select_sizes(ctx, n, vocab, masked):
    select_case(ctx, np.random.default_rng(vocab), n, vocab, masked=masked, history=min(vocab * 2, 300))


@pytest.mark.parametrize("kw", [{"in_place": True}, {"pad": 3}, {"pad": 4, "mask_pad": 2}, {"shift": 1}, {"spans": 1},
                                {"spans": 8}, {"history": 0}, {"biases": 0}, {"want_out": False}, {"want_tokens": False},
                                {"make": edges}, {"make": edges, "in_place": True, "pad": 1}, {"ids": [3] * 5000},
                                {"shift": 3, "pad": 5, "in_place": True}])
def test_select_options(ctx, kw):
    select_case(ctx, np.random.default_rng(11), 4, 700, **kw)


@pytest.mark.parametrize("pen", [(65536, 0, 0), (0, 0, 0), (-5, 70000, 0), (1, 0, 0), (I32_MAX, I32_MAX, I32_MAX),
                                 (I32_MIN, I32_MIN, I32_MIN), (32768, 0, -65536)])
@pytest.mark.parametrize("make", [acts, edges])
def test_select_penalties(ctx, pen, make):
    select_case(ctx, np.random.default_rng(12), 3, 200, history=400, penalties=np.array([pen] * 3, dtype=np.int32), make=make)


def test_select_without_rules_is_argmax_first(ctx):
    rng = np.random.default_rng(13)
    for n, vocab in [(1, 262144), (3, 5000), (2, 7)]:
        x = rng.integers(-50, 51, size=(n, vocab)).astype(np.int32)  # (many ties)
        x[0, :] = I32_MIN if vocab == 7 else x[0, :]
        xb, tb = ctx.to_device(x), ctx.empty(n, np.uint32)
        ctx.select_tokens(xb, n, vocab, vocab, None, None, 0, tb)
        assert tb.numpy().tolist() == x.argmax(1).tolist()
        assert int(tb.numpy()[0]) == ctx.argmax_first(xb, vocab)


@pytest.mark.parametrize("history,biases", [(2048, 0), (2049, 400), (7000, 700), (0, 900)])
def test_select_long_rules(ctx, history, biases):
    # histories and biases of more entries than a workgroup holds at a time
    select_case(ctx, np.random.default_rng(history + biases), 2, 9000, history=history, biases=biases)


def test_select_allowed_minimum_is_chosen_over_nothing(ctx):
    # the only allowed token holds the lowest value; masked ones hold it as well
    x = np.full((2, 100), I32_MIN, dtype=np.int32)
    x[1] = 5
    mask = np.zeros((2, 4), dtype=np.uint32)
    mask[0, 2] = 1 << 5
    tb = ctx.empty(2, np.uint32)
    out = ctx.empty((2, 100))
    ctx.select_tokens(ctx.to_device(x), 2, 100, 100, rd.LogitRules(mask=ctx.to_device(mask), mask_stride=4), out, 100, tb)
    assert tb.numpy().tolist() == [69, rd.DET_NO_TOKEN]
    assert (out.numpy() == I32_MIN).all()


def test_select_cuts_spans_and_biases_at_their_arrays(ctx):
    # device words past the arrays select nothing past them
    x = np.zeros((1, 64), dtype=np.int32)
    ids, pen = np.array([1, 2, 2], dtype=np.uint32), np.array([[65536, 65536, 0]], dtype=np.int32)
    spans = np.array([[[1, 2**32 - 1], [5, 9]]], dtype=np.uint32)
    begin, bi, bv = np.array([0, 4000], dtype=np.uint32), np.array([2, 63], np.uint32), np.array([65536, 9], np.int32)
    out, tb = ctx.empty((1, 64)), ctx.empty(1, np.uint32)
    rules = rd.LogitRules(penalties=ctx.to_device(pen), ids=ctx.to_device(ids), n_ids=3, spans=ctx.to_device(spans),
                          spans_per_row=2, bias_begin=ctx.to_device(begin), bias_ids=ctx.to_device(bi),
                          bias_values=ctx.to_device(bv), n_bias=2)
    ctx.select_tokens(ctx.to_device(x), 1, 64, 64, rules, out, 64, tb)
    exp = np.zeros(64, dtype=np.int32)
    exp[2], exp[63] = -65536, 9
    assert np.array_equal(out.numpy()[0], exp) and tb.numpy()[0] == 63


@pytest.mark.parametrize("begin", [2**32 - 1, 2**32 - 3, 2**32 - 515, 9, 2])
def test_select_biases_that_begin_past_their_end(ctx, begin):
    x = np.zeros((1, 40), dtype=np.int32)
    rules = rd.LogitRules(bias_begin=ctx.to_device(np.array([begin, 2], dtype=np.uint32)),
                          bias_ids=ctx.to_device(np.array([3, 7], dtype=np.uint32)),
                          bias_values=ctx.to_device(np.array([5, 6], dtype=np.int32)), n_bias=2)
    out = ctx.empty((1, 40))
    ctx.select_tokens(ctx.to_device(x), 1, 40, 40, rules, out, 40, None)
    assert not out.numpy().any()


def test_select_refusals(ctx):
    x, tb = ctx.empty((2, 64)), ctx.empty(2, np.uint32)
    pen = ctx.to_device(np.zeros(6, np.int32))
    ok = (x, 2, 64, 64, None, x, 64, tb)
    for status, args in [(2, (x, 2, 0, 64, None, x, 64, tb)), (1, (None,) + ok[1:]), (1, (x, 65536) + ok[2:]),
                         (1, (x, 2, 64, 63, None, x, 64, tb)), (1, (x, 2, 64, 64, None, x, 63, tb)),
                         (1, (x, 2, 64, 64, None, x, 65, tb)), (1, (x, 2, 64, 64, None, None, 0, None)),
                         (1, (x, 2, 64, 64, rd.LogitRules(mask=x, mask_stride=1), x, 64, tb)),
                         (1, (x, 2, 64, 64, rd.LogitRules(penalties=pen, n_ids=2, ids=x), x, 64, tb)),
                         (1, (x, 2, 64, 64, rd.LogitRules(penalties=pen, n_ids=2, spans=x), x, 64, tb)),
                         (1, (x, 2, 64, 64, rd.LogitRules(penalties=pen, n_ids=2, ids=x, spans=x, spans_per_row=9), x, 64, tb)),
                         (1, (x, 2, 64, 64, rd.LogitRules(bias_begin=x, n_bias=2), x, 64, tb)),
                         (1, (x, 2, 64, 64, rd.LogitRules(bias_begin=x, bias_ids=x, bias_values=x, n_bias=2**28 + 1), x, 64, tb))]:
        with pytest.raises(rd.DetError) as e:
            ctx.select_tokens(*args)
        assert e.value.status == status, args
    ctx.select_tokens(*ok)
    ctx.select_tokens(None, 0, 64, 64, None, None, 64, None)


# ---------------------------------------------------------------------------
# Together: one verification step, eager and as a recorded graph
# ---------------------------------------------------------------------------
class Step:
    """The chain of one layer-less verification step: fused q/k/v projection with the requests' adapters, head norms
    with the tree's positions, tree attention, output projection with adapters to logits, decoding rules."""

    hidden, heads, kv_heads, hd, vocab = 96, 4, 2, 32, 700

    def __init__(self, ctx, rng, cached, parents):
        self.ctx, self.cached = ctx, cached
        self.drafts = [len(p) for p in parents]
        m = self.m = sum(self.drafts)
        self.qw, self.kw = self.heads * self.hd, self.kv_heads * self.hd
        width = self.qw + 2 * self.kw
        self.w_qkv, self.w_out = weights(rng, width, self.hidden, "int8"), weights(rng, self.vocab, self.qw, "i16")
        self.ads = [[(weights(rng, r, c, k), weights(rng, rows, r, k), 40000 + 9000 * r) for r, k in ((4, "int8"), (20, "i16"))]
                    for rows, c in ((width, self.hidden), (self.vocab, self.qw))]
        self.index = np.repeat([0, 5, 1][:len(parents)], self.drafts).astype(np.uint32)
        masks, depths = zip(*(rd.tree_masks(p) for p in parents))
        self.masks = np.concatenate(masks)
        self.positions = np.concatenate([n + d for n, d in zip(cached, depths)]).astype(np.uint32)
        self.gain = 65536 + acts(rng, self.hd, std=0.1)
        self.kc, self.vc = ([acts(rng, n, self.kw) for n in cached] for _ in range(2))
        self.pen = np.array([[72090, 6553, 3000]] * m, dtype=np.int32)
        self.ids = rng.integers(0, self.vocab, size=60).astype(np.uint32)
        self.spans = np.array([[[3 * i, 3 * i + 20]] for i in range(m)], dtype=np.uint32)
        self.bits = rng.integers(0, 2**32, size=(m, 22), dtype=np.uint64).astype(np.uint32)
        d = ctx.to_device
        self.table = rd.RopeTable(ctx, 16, 16, 10000 * ONE, layout=rd.DET_ROPE_INTERLEAVED)
        self.mat = [ctx.upload_matrix(w[0], w[1]) for w in (self.w_qkv, self.w_out)]
        self.sets = [rd.Adapters(ctx, rows, c, [rd.Adapter(a[0], b[0], s, down_scale=a[1], up_scale=b[1]) for a, b, s in ads])
                     for ads, rows, c in zip(self.ads, (width, self.vocab), (self.hidden, self.qw))]
        self.x, self.idx, self.pos, self.mask = ctx.empty((m, self.hidden)), d(self.index), d(self.positions), d(self.masks)
        self.qkv, self.attn = ctx.empty((m, width)), ctx.empty((m, self.qw))
        self.logits, self.tokens = ctx.empty((m, self.vocab)), ctx.empty(m, np.uint32)
        self.gb = d(self.gain)
        self.heads_sets = [rd.HeadRows(At(self.qkv, 0), width, self.heads, gain=self.gb),
                           rd.HeadRows(At(self.qkv, self.qw), width, self.kv_heads, gain=self.gb),
                           rd.HeadRows(At(self.qkv, self.qw + self.kw), width, self.kv_heads, rotate=False)]
        self.kept = [(d(k), d(v)) for k, v in zip(self.kc, self.vc)]
        self.views = rd.attn_caches([rd.AttnCache(k, v, self.kw, n) for (k, v), n in zip(self.kept, cached)])
        self.counts = rd.u32_array(self.drafts)
        self.rules = rd.LogitRules(penalties=d(self.pen), ids=d(self.ids), n_ids=60, spans=d(self.spans),
                                   mask=d(self.bits), mask_stride=22)
        self.width = width

    def run(self):
        c, w = self.ctx, self.width
        c.det_linear_adapters(self.mat[0], self.sets[0], self.m, self.x, self.idx, self.qkv)
        c.head_norm_rope(self.table, self.pos, self.m, self.hd, 4295, self.heads_sets)
        c.attention_tree(self.views, self.counts, At(self.qkv, 0), w, At(self.qkv, self.qw),
                         At(self.qkv, self.qw + self.kw), w, self.mask, None, self.heads, self.kv_heads, self.hd,
                         self.attn, self.qw)
        c.det_linear_adapters(self.mat[1], self.sets[1], self.m, self.attn, self.idx, self.logits)
        c.select_tokens(self.logits, self.m, self.vocab, self.vocab, self.rules, self.logits, self.vocab, self.tokens)

    def expected(self, x):
        bits = [[(a[2], b[2], s) for a, b, s in ads] for ads in self.ads]
        y = ref.linear_adapters(self.w_qkv[2], bits[0], x, self.index)
        freq, at, n = ref.frequencies(10000 * ONE, 16, 8), 0, self.heads + 2 * self.kv_heads
        for r in range(self.m):
            for h in range(n):
                c = slice(h * self.hd, (h + 1) * self.hd)
                rotate = h < self.heads + self.kv_heads
                y[r, c] = ref.head_row(y[r, c], self.gain if rotate else None, 4295, True, freq, int(self.positions[r]), 1,
                                       65536, rotate)
        o = ref.attention_tree(list(zip(self.kc, self.vc)), self.drafts, y[:, :self.qw], y[:, self.qw:self.qw + self.kw],
                               y[:, self.qw + self.kw:], self.masks, None, self.heads, self.kv_heads, self.hd)
        z = ref.linear_adapters(self.w_out[2], bits[1], o, self.index)
        return ref.select(z, self.pen, self.ids, [[tuple(map(int, s)) for s in r] for r in self.spans], None, self.bits)


def test_verification_step_eager_and_recorded(ctx):
    rng = np.random.default_rng(21)
    step = Step(ctx, rng, [90, 0, 33], [[-1, 0, 0, 1], [-1], [-1, -1, 1]])
    inputs = [acts(rng, step.m, step.hidden) for _ in range(3)]
    want = [step.expected(x) for x in inputs]

    def check(x, exp):
        assert np.array_equal(step.logits.numpy(), exp[0])
        assert np.array_equal(step.tokens.numpy(), exp[1])

    for x, exp in zip(inputs, want):
        step.x.upload(x)
        step.run()
        check(x, exp)
    graph = ctx.capture(step.run)
    other = Step(ctx, np.random.default_rng(22), [40], [[-1, 0]])
    for turn in range(3):
        for x, exp in zip(inputs, want):
            step.x.upload(x)
            graph.launch()
            check(x, exp)
            other.x.upload(inputs[0][:other.m])
            # eager work between the replays; a larger call replaces the shared scratch
            ctx.select_tokens(step.logits, 1, 700, 700, None, None, 0, step.tokens)
            if turn == 1:
                big = ctx.empty((64, 40000))
                ctx.select_tokens(big, 64, 40000, 40000, None, big, 40000, ctx.empty(64, np.uint32))


def test_two_contexts_at_once():
    a, b = rd.Context(0), rd.Context(0)
    rng = np.random.default_rng(23)
    steps = [Step(c, rng, [70, 5], [[-1, 0, 1], [-1, -1]]) for c in (a, b)]
    for s in steps:
        s.index[:] = 0
        s.idx.upload(s.index)
    xs = [acts(rng, s.m, s.hidden) for s in steps]
    for s, x in zip(steps, xs):
        s.x.upload(x)
    for _ in range(20):
        for s in steps:
            s.run()
    for s, x in zip(steps, xs):
        exp = s.expected(x)
        assert np.array_equal(s.logits.numpy(), exp[0]) and np.array_equal(s.tokens.numpy(), exp[1])
    a.close()
    b.close()


def test_captures_refuse_scratch_that_would_grow():
    c = rd.Context(0)
    x, tb = c.empty((2, 9000)), c.empty(2, np.uint32)
    with pytest.raises(rd.DetError) as e:
        c.capture(lambda: c.select_tokens(x, 2, 9000, 9000, None, None, 0, tb))
    assert e.value.status == 1 and "grow" in str(e.value)
    c.select_tokens(x, 2, 9000, 9000, None, None, 0, tb)
    g = c.capture(lambda: c.select_tokens(x, 2, 9000, 9000, None, None, 0, tb))
    g.launch()
    assert tb.numpy().tolist() == np.argmax(x.numpy(), 1).tolist()
    with pytest.raises(rd.DetError):
        c.capture(lambda: rd.RopeTable(c, 4, 4, ONE))
    c.close()
