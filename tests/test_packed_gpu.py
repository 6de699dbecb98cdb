"""The packed-batch operators on the GPU against their definitions in 64 bits
(tests/packed_reference.py), with bounds derived there from the arithmetic:
row maps, rotary positions with several axes, and attention with capped
scores, distance bias and document, causal and prefix masks."""
import numpy as np
import pytest

import packed_reference as ref

pytestmark = pytest.mark.gpu


def _status():
    import torch
    import beatlm_b200 as bl
    torch.cuda.synchronize()
    st = bl.status(reset=True)
    return st.code


# ------------------------------------------------------------------ row maps

def _pack(grids, capacity, lead=0, normalized=False, positions=True):
    import torch
    from beatlm_b200 import ops
    g = torch.tensor(grids, dtype=torch.int32, device="cuda").reshape(-1, 3)
    off = torch.full((len(grids) + 1,), -7, dtype=torch.int32, device="cuda")
    img = torch.full((capacity,), -7, dtype=torch.int32, device="cuda")
    pos = torch.full((capacity, 3), -7.0, device="cuda") if positions else None
    ops.pack(g, offsets=off, image=img, positions=pos, lead=lead, normalized=normalized)
    return off.cpu().numpy(), img.cpu().numpy(), pos.cpu().numpy() if positions else None


@pytest.mark.parametrize("grids,capacity,lead", [
    ([(1, 1, 1)], 1, 0), ([(1, 1, 1)], 5, 2), ([(1, 37, 37), (1, 18, 25), (4, 7, 3)], 1922, 1),
    ([(1, 3, 4), (0, 5, 5), (1, -2, 3), (2, 2, 2)], 31, 3),
    ([(0, 1, 1), (1, 2, 3), (1, 1, 0)], 9, 0), ([(0, 0, 0)], 7, 4)])
@pytest.mark.parametrize("normalized", [False, True])
def test_pack_matches_the_definition(grids, capacity, lead, normalized):
    off, img, pos = _pack(grids, capacity, lead, normalized)
    woff, wimg, wpos = ref.pack(grids, capacity, lead, normalized)
    assert np.array_equal(off, woff) and np.array_equal(img, wimg)
    assert np.all(np.abs(pos - wpos) <= np.abs(wpos) * ref.EPS["f32"])  # one division
    assert _status() == 0


@pytest.mark.parametrize("images", [31, 32, 33, 255, 257, 1024, 1025, 2500, 4096, 4097])
def test_pack_of_many_images(images):
    rng = np.random.default_rng(images)
    grids = [tuple(int(v) for v in g) for g in rng.integers(0, 6, (images, 3))]
    total = sum(t * h * w + 2 for t, h, w in grids if min(t, h, w) > 0)
    off, img, pos = _pack(grids, total + 3, 2)
    woff, wimg, wpos = ref.pack(grids, total + 3, 2, False)
    assert np.array_equal(off, woff) and np.array_equal(img, wimg) and np.array_equal(pos, wpos)


@pytest.mark.parametrize("normalized", [False, True])
@pytest.mark.parametrize("shape", [(1, 2100, 2003), (3, 1, 1400001), (1, 1, 2 ** 22 + 5)])
def test_pack_of_more_rows_than_24_bits_hold_exactly(shape, normalized):
    """Row numbers and sides past 2^22, where places leave the f32 path."""
    import torch
    t, h, w = shape
    rows = t * h * w
    off, img, pos = _pack([shape], rows, 0, normalized)
    r = torch.arange(rows)
    c = torch.stack([r // (h * w), r // w % h, r % w], 1).double()
    n = torch.tensor(shape).double()
    want = ((2 * c + 1 - n) / n if normalized else c).numpy()
    assert np.all(np.abs(pos - want) <= np.abs(want) * ref.EPS["f32"])  # one division
    assert (img == 0).all() and list(off) == [0, rows]


@pytest.mark.parametrize("grids,capacity", [
    ([(1, 4, 4), (1, 4, 4), (1, 4, 4)], 20), ([(1, 5, 5)], 7),
    ([(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1), (1, 2, 2)], 40),
    ([(1, 2, 2), (1, 65536, 65536), (3, 3, 3)], 33)])
def test_pack_cuts_off_at_the_capacity_and_says_so(grids, capacity):
    off, img, pos = _pack(grids, capacity, 1)
    count = 0
    for i, g in enumerate(grids):
        lo, count = count, min(capacity, count + 1 + int(np.prod([int(v) for v in g], dtype=object)))
        assert off[i] == lo and off[i + 1] == count
        assert np.all(img[lo:count] == i)
    assert _status() == 0x50


def test_pack_without_maps_writes_the_offsets_alone():
    import torch
    from beatlm_b200 import ops
    g = torch.tensor([[1, 2, 3], [1, 4, 4]], dtype=torch.int32, device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    ops.pack(g, offsets=off, capacity=100)
    assert off.tolist() == [0, 6, 22]
    img = torch.full((25,), -7, dtype=torch.int32, device="cuda")
    ops.pack(g, offsets=off, image=img[:23])
    assert img[:23].tolist() == [0] * 6 + [1] * 16 + [-1] and img[23:].tolist() == [-7, -7]
    pos = torch.full((24, 3), -7.0, device="cuda")
    ops.pack(g, offsets=off, positions=pos[1:24])  # positions at an odd address
    assert pos[0].tolist() == [-7.0] * 3 and pos[2].tolist() == [0.0, 0.0, 1.0]


# ------------------------------------------------------------------ rotary

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _torch_dtype(name):
    import torch
    return getattr(torch, DT[name])


def _check_rope(got, x, pos, sections, dtype, **kw):
    want, off = ref.rope(x.double().cpu().numpy(), pos.double().cpu().numpy(), sections, **kw)
    got = got.double().cpu().numpy()
    bound = off * (1 + ref.EPS[dtype]) + np.abs(want) * ref.EPS[dtype]
    if dtype == "f16":
        bound = bound + 2.0 ** -25  # half the least step below the normal range
    bad = np.abs(got - want) > bound
    assert not bad.any(), (np.argwhere(bad)[:3], np.abs(got - want).max())


@pytest.mark.parametrize("pairing", ["half", "adjacent", "axis_half"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,heads,head_dim,sections", [
    (1, 1, 2, (1,)), (1, 32, 64, (10, 11, 11)), (7, 3, 64, (16, 16)), (33, 12, 64, (32,)),
    (5, 2, 80, (20, 20)), (9, 5, 72, (36,)), (17, 1, 96, (8, 16, 24)), (3, 4, 128, (64,)),
    (2, 3, 256, (42, 43, 43)), (6, 2, 34, (8, 9)), (130, 9, 64, (16, 16))])
def test_rope_matches_the_definition(rows, heads, head_dim, sections, dtype, pairing):
    import torch
    from beatlm_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(rows * heads)
    x = torch.randn((rows, heads, head_dim), generator=g, device="cuda").to(_torch_dtype(dtype))
    pos = (torch.rand((rows, len(sections)), generator=g, device="cuda") * 2e5 - 1e5)
    pos[::2] = pos[::2].round()
    for inverse in (False, True):
        y = ops.rope(x, pos, sections=sections, theta=10000.0, pairing=pairing, inverse=inverse,
                     out=torch.full_like(x, 9.0))
        _check_rope(y, x, pos, sections, dtype, theta=10000.0, pairing=pairing, inverse=inverse)


def test_rope_leaves_what_does_not_turn():
    import torch
    from beatlm_b200 import ops
    x = torch.randn((11, 3, 64), device="cuda").to(torch.bfloat16)
    pos = torch.rand((11, 2), device="cuda") * 30
    y = ops.rope(x, pos, sections=(8, 8), out=torch.full_like(x, 9.0))
    assert torch.equal(y[..., 32:], x[..., 32:])
    _check_rope(y[..., :32], x[..., :32], pos, (8, 8), "bf16", theta=100.0, pairing="half",
                inverse=False)
    z = x.clone()
    assert ops.rope(z, pos, sections=(8, 8)) is z and torch.equal(z, y)  # in place: the same bits
    still = ops.rope(x, torch.zeros((11, 2), device="cuda"), sections=(16, 16),
                     out=torch.empty_like(x))
    assert torch.equal(still, x)  # position zero: class and register tokens


@pytest.mark.parametrize("qk", ["f16", "bf16"])
def test_rope_turns_q_and_k_of_packed_rows_in_place(qk):
    import torch
    from beatlm_b200 import ops
    rows, heads, kv = 21, 4, 2
    packed = ops.pack_qkv(np.random.default_rng(3).standard_normal((rows, 3, 4, 64)), qk)
    qkv = packed.reshape(rows, 12 * 64)[:, :(heads + 2 * kv) * 64]  # rows 12 heads apart
    before = qkv.clone()
    grid = torch.stack([torch.arange(rows, device="cuda") // 5,
                        torch.arange(rows, device="cuda") % 5], 1).float()
    pos = torch.zeros((rows, 3), device="cuda")
    pos[:, 1:] = grid
    ops.rope(qkv, pos[:, 1:], sections=(16, 16), heads=heads + kv, head_dim=64, dtype=qk)
    turned = (heads + kv) * 64
    assert torch.equal(qkv[:, turned:], before[:, turned:])  # V stays
    t = _torch_dtype(qk)
    x = before[:, :turned].view(t).reshape(rows, heads + kv, 64)
    _check_rope(qkv[:, :turned].view(t).reshape(x.shape), x, grid, (16, 16), qk, theta=100.0,
                pairing="half", inverse=False)


def test_rope_ladders_and_given_frequencies():
    import torch
    from beatlm_b200 import ops
    x = torch.randn((40, 2, 64), device="cuda")
    pos = torch.rand((40, 3), device="cuda") * 4 - 2
    y = ops.rope(x, pos, sections=(16, 8, 8), theta=500.0, shared=True, out=torch.empty_like(x))
    _check_rope(y, x, pos, (16, 8, 8), "f32", theta=500.0, pairing="half", inverse=False,
                shared=True)
    freqs = [0.1 * (i + 1) for i in range(32)]
    y = ops.rope(x, pos, sections=(16, 8, 8), freqs=freqs, out=torch.empty_like(x))
    _check_rope(y, x, pos, (16, 8, 8), "f32", theta=1.0, pairing="half", inverse=False,
                freqs=freqs)


@pytest.mark.parametrize("pairing", ["half", "adjacent", "axis_half"])
def test_the_inverse_rotation_is_the_gradient(pairing):
    """sum(w * rope(x)) changes with x as the inverse rotation of w says: the
    formula's gradient, and differences of the forward pass (linear in x, so a
    difference of any step is exact but for f32 rounding: 64 products of values
    below 8, each off by 2^-23 of 8, and sums)."""
    import torch
    from beatlm_b200 import ops
    kw = dict(sections=(12, 20), theta=50.0, pairing=pairing)
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = (torch.randn((4, 2, 64), generator=g, device="cuda") for _ in range(2))
    pos = torch.rand((4, 2), generator=g, device="cuda") * 9
    grad = ops.rope(w, pos, inverse=True, out=torch.empty_like(w), **kw)
    _check_rope(grad, w, pos, kw["sections"], "f32", theta=50.0, pairing=pairing, inverse=True)
    fwd = lambda t: (ops.rope(t, pos, out=torch.empty_like(t), **kw).double() * w.double()).sum()  # noqa: E731
    for at in [(0, 0, 0), (1, 1, 13), (2, 0, 33), (3, 1, 63)]:
        up, down = x.clone(), x.clone()
        up[at], down[at] = x[at] + 2.0, x[at] - 2.0
        diff = (fwd(up) - fwd(down)) / (up[at].double() - down[at].double())
        assert abs(float(diff) - float(grad[at])) <= 128 * 8 * 2.0 ** -23


@pytest.mark.parametrize("pairing", ["half", "adjacent", "axis_half"])
def test_cosines_and_sines_are_good_to_their_own_size(pairing):
    """Pairs (1, 0) turn to (cos, sin) themselves: each within 2 ulp (the function),
    half a one (its correction for what the angle's 32 bits left out) and the 64-bit
    angle's own error, small sines of angles near a half turn too."""
    import torch
    from beatlm_b200 import ops
    rows, sections = 1500, (16, 16)
    g = torch.Generator(device="cuda").manual_seed(77)
    pos = torch.rand((rows, 2), generator=g, device="cuda") * 2000 - 1000
    x = torch.zeros((rows, 1, 64), device="cuda")
    lows = [lo for _, _, lo, _ in ref.pairs(64, sections, pairing)]
    x[:, :, lows] = 1.0
    got = ops.rope(x, pos, sections=sections, theta=100.0, pairing=pairing, out=torch.empty_like(x))
    want, _ = ref.rope(x.double().cpu().numpy(), pos.double().cpu().numpy(), sections, 100.0,
                       pairing, False)
    size = np.maximum(np.abs(want), 2.0 ** -100)
    ulp = 2.0 ** (np.floor(np.log2(size)) - 23)
    bound = 2.5 * ulp * (1 + 2.0 ** -20) + 1000 * 2.0 ** -50 + 2.0 ** -43
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound), (off / bound).max()


# ------------------------------------------------------------------ attention

class Case:
    """Random packed rows with NaN wherever a sequence has ended."""

    def __init__(self, lens, heads=2, kv=None, qk="bf16", form="packed", tokens=None, seed=0,
                 gap=9, std=1.0, extra=0):
        import torch
        self.heads, self.kv, self.qk = heads, kv or heads, qk
        kv, lens = self.kv, list(lens)
        rng = np.random.default_rng(seed + sum(lens) + heads)
        if form == "packed":
            offsets = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            rows = int(offsets[-1]) + gap
            self.where = ref.spans(len(lens), rows, offsets=offsets)
            self.kw = {"offsets": torch.from_numpy(offsets).cuda()}
        else:
            tokens = tokens or max(lens)
            rows = tokens * len(lens)
            self.where = ref.spans(len(lens), tokens, lengths=lens)
            self.kw = {"lengths": torch.tensor(lens, dtype=torch.int32).cuda()}
        live = np.zeros(max(rows, 1), bool)
        for b, e in self.where:
            live[b:e] = True
        x = rng.standard_normal((live.size, heads + 2 * kv, 64), dtype=np.float32) * std
        x[~live] = np.nan
        t = torch.bfloat16 if qk == "bf16" else torch.float16
        x = torch.from_numpy(x)
        qkp, v = x[:, :heads + kv].to(t), x[:, heads + kv:].to(torch.float16)
        buf = torch.full((live.size, heads + 2 * kv + extra, 64), -1, dtype=torch.int16)
        buf[:, :heads + kv], buf[:, heads + kv:heads + 2 * kv] = qkp.view(torch.int16), v.view(torch.int16)
        self.buf = buf.cuda()
        self.qkv = self.buf[:, :heads + 2 * kv]
        self.q, self.k = qkp[:, :heads].double().numpy(), qkp[:, heads:].double().numpy()
        self.v = v.double().numpy()
        self.rows = live.size

    def run(self, out_dtype="bf16", out=None, **kw):
        import torch
        from beatlm_b200 import ops
        if out is None:
            out = torch.full((self.rows, self.heads * 64), 7.0, device="cuda",
                             dtype=_torch_dtype(out_dtype))
        for name in ("slopes", "positions", "prefix"):
            if kw.get(name) is not None:
                kw[name] = torch.as_tensor(np.asarray(kw[name], np.int32 if name == "prefix"
                                                      else np.float32)).cuda()
        return ops.masked_attention(self.qkv, heads=self.heads, kv_heads=self.kv, qk_dtype=self.qk,
                                    out=out, **{**self.kw, **kw})

    def check(self, out, out_dtype="bf16", **kw):
        kw.pop("key_splits", None)
        want, off, written = ref.attention(self.q, self.k, self.v, self.where, **kw)
        got = out.double().cpu().numpy().reshape(self.rows, -1)[:, :self.heads * 64]
        got = got.reshape(self.rows, self.heads, 64)
        assert np.all(got[~written] == 7.0), "rows that were not asked for were written"
        got, want, off = got[written], want[written], off[written]
        assert np.isfinite(got).all()
        bound = off * (1 + ref.EPS[out_dtype]) + np.abs(want) * ref.EPS[out_dtype] + 2.0 ** -25
        bad = np.abs(got - want) > bound
        assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want)[bad].max(),
                               bound[bad].min())
        assert _status() == 0

    def both(self, out_dtype="bf16", **kw):
        self.check(self.run(out_dtype, **kw), out_dtype, **kw)


SLOPES = [0.5, 0.25, 0.125, 0.0625, 0.03, 0.01, 0.7, 1.5]


@pytest.mark.parametrize("n", [1, 2, 31, 63, 64, 65, 127, 128, 129, 191, 192, 193, 300, 777])
@pytest.mark.parametrize("mask", [None, "causal"])
def test_attention_of_one_sequence(n, mask):
    Case([n], heads=3).both(mask=mask)


@pytest.mark.parametrize("qk,out_dtype", [("f16", "f32"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("heads,kv", [(4, 4), (4, 2), (6, 1)])
def test_attention_types_and_grouped_heads(qk, out_dtype, heads, kv):
    Case([70, 1, 200], heads=heads, kv=kv, qk=qk, seed=5).both(out_dtype)


@pytest.mark.parametrize("lens", [[0], [5, 0, 0, 130, 0], [1] * 70, [64] * 5, [128, 128],
                                  [257, 3, 64, 65], [0] * 40 + [33] + [0] * 40])
@pytest.mark.parametrize("mask", [None, "causal", "prefix"])
def test_document_masks_never_leak(lens, mask):
    kw = {"prefix": [(7 * i) % (n + 3) for i, n in enumerate(lens)]} if mask == "prefix" else {}
    Case(lens, seed=11).both(mask=mask, **kw)


def test_many_short_documents():
    rng = np.random.default_rng(2)
    Case([int(n) for n in rng.integers(0, 9, 700)], heads=1).both(mask="causal")


@pytest.mark.parametrize("prefix", [-5, 0, 1, 63, 64, 65, 200, 10 ** 6])
def test_prefix_lengths(prefix):
    Case([200, 66], seed=3).both(mask="prefix", prefix=[prefix, prefix])


@pytest.mark.parametrize("cap,std", [(30.0, 1.0), (5.0, 3.0), (0.5, 6.0), (50.0, 0.1)])
@pytest.mark.parametrize("mask", [None, "causal"])
def test_capped_scores(cap, std, mask):
    Case([150, 33], seed=9, std=std).both(cap=cap, mask=mask)


@pytest.mark.parametrize("last", [0, 1])
@pytest.mark.parametrize("cap", [1e6, 1e12, 1e30])
def test_a_cap_far_above_the_scores_is_none(cap, last):
    # cap tanh(s / cap) is s less s^3 / (3 cap^2), below 1e-8 here: held to the uncapped bound
    c = Case([150, 33], heads=2, seed=19)
    c.check(c.run(cap=cap, last_rows=last), last_rows=last)


@pytest.mark.parametrize("last", [1, 40])
def test_a_capped_tile_with_one_score_far_below(last):
    """Keys near -cap / 2 beside ordinary ones, which keep their own precision."""
    import torch
    c = Case([200], heads=1, qk="f16", seed=23)
    for j, by in ((5, 6000.0), (70, 6250.0), (140, 6500.0)):
        c.qkv[j, 1] = (c.qkv[199, 0].view(torch.float16) * -by).view(torch.int16)
    c.k = c.qkv.view(torch.float16).double().cpu().numpy()[:, 1:2]
    # (the keys near -cap / 2 have no weight in the last row, those of thousands all of it in
    # the others, capped or not)
    c.check(c.run(cap=1e5, last_rows=last), last_rows=last)


@pytest.mark.parametrize("axes", [0, 1, 2, 3])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_distance_bias(axes, cap):
    c = Case([140, 67], heads=4, kv=2, seed=axes)
    pos = None
    if axes:
        pos = np.random.default_rng(axes).integers(0, 30, (c.rows, axes)).astype(np.float64)
    c.both(slopes=np.array(SLOPES[:4], np.float32), positions=pos, cap=cap)


def test_distance_bias_of_far_rows_and_signs():
    c = Case([90], heads=2)
    pos = np.zeros((c.rows, 2))
    pos[:, 0] = 1e5 + np.arange(c.rows) * 3
    c.both(slopes=np.array([-0.01, 2.0], np.float32), positions=pos)
    c.both(slopes=np.array([-0.01, 2.0], np.float32), mask="causal")


@pytest.mark.parametrize("last", [1, 2, 3, 4, 5, 64, 129, 10 ** 6])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1), (3, 1), (8, 1)])
def test_last_rows_of_padded_sequences(last, heads, kv):
    c = Case([300, 1, 0, 77, 129], heads=heads, kv=kv, form="padded", tokens=310, seed=last % 97)
    c.both(mask="causal", last_rows=last)
    c.both(last_rows=last, cap=25.0, slopes=np.array(SLOPES[:heads], np.float32))


@pytest.mark.parametrize("last", [1, 40])
def test_last_rows_of_packed_sequences(last):
    Case([100, 0, 3, 500], heads=4, kv=2, seed=8).both(mask="prefix", prefix=[10, 0, 9, 50],
                                                       last_rows=last)


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("last", [0, 1, 100])
def test_key_splits(splits, last):
    c = Case([700, 20, 129], heads=2, seed=4)
    kw = dict(mask="causal", last_rows=last, key_splits=splits,
              slopes=np.array(SLOPES[:2], np.float32))
    c.both(**kw)
    assert np.array_equal(c.run(**kw).float().cpu().numpy(), c.run(**kw).float().cpu().numpy())


def _places(c, axes, seed):
    """Places of a case's rows on a grid, some of them off it; NaN behind its sequences."""
    rng = np.random.default_rng(seed)
    pos = rng.integers(0, 40, (c.rows, axes)).astype(np.float64)
    pos[::3] += rng.random((c.rows, axes))[::3]
    dead = np.ones(c.rows, bool)
    for b, e in c.where:
        dead[b:e] = False
    pos[dead] = np.nan
    return pos.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("mask", [None, "causal", "prefix"])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("last", [0, 1, 4, 40])
def test_places_under_masks_and_of_newest_rows(axes, mask, cap, last):
    """Few rows (up to 16 a K/V head) and tiles; prefixes that end inside one."""
    lens = [300, 0, 67, 1, 129]
    c = Case(lens, heads=4, kv=2, seed=axes, form="padded" if axes == 2 else "packed")
    kw = {"prefix": [100, 3, 70, 0, 65]} if mask == "prefix" else {}
    c.both(slopes=np.array(SLOPES[:4], np.float32), positions=_places(c, axes, axes), cap=cap,
           mask=mask, last_rows=last, **kw)


@pytest.mark.parametrize("splits", [2, 3, 8])
@pytest.mark.parametrize("last", [0, 1, 100])
@pytest.mark.parametrize("cap,axes", [(20.0, None), (20.0, 0), (None, 2), (2.0, 3)])
def test_key_splits_with_caps_and_places(splits, last, cap, axes):
    c = Case([700, 20, 129], heads=2, seed=4)
    kw = dict(mask="causal", last_rows=last, key_splits=splits, cap=cap)
    if axes is not None:
        kw["slopes"] = np.array(SLOPES[3:5], np.float32)
    if axes:
        kw["positions"] = _places(c, axes, 9)
    c.both(**kw)


@pytest.mark.parametrize("form", ["packed", "padded"])
@pytest.mark.parametrize("last", [1, 20])
def test_newest_rows_of_many_sequences(form, last):
    rng = np.random.default_rng(last)
    for batch in (32, 33, 70):
        lens = [int(v) for v in rng.integers(0, 500, batch)]
        c = Case(lens, heads=2, kv=1, form=form, tokens=512, seed=batch)
        c.both(mask="causal", last_rows=last, slopes=np.array(SLOPES[:2], np.float32))


@pytest.mark.parametrize("batch", [2, 31, 32, 33])
@pytest.mark.parametrize("form", ["packed", "padded"])
@pytest.mark.parametrize("mask", [None, "causal", "prefix"])
@pytest.mark.parametrize("last", [0, 150])
def test_every_tile_of_a_ragged_batch_is_found(batch, form, mask, last):
    """Tiles are ranked by their keys up to 32 sequences, walked beyond."""
    rng = np.random.default_rng(batch + last)
    lens = [int(v) for v in rng.integers(0, 400, batch)]
    lens[0], lens[-1] = 385, 0
    kw = {"prefix": [int(v) for v in rng.integers(0, 400, batch)]} if mask == "prefix" else {}
    Case(lens, heads=1, form=form, seed=batch).both(mask=mask, last_rows=last, **kw)


@pytest.mark.parametrize("lens,heads,form", [
    ([1500, 200, 64, 900], 2, "packed"), ([1500, 200, 0, 900], 2, "padded"),
    ([1600, 300], 5, "padded"), ([1600, 1000], 5, "packed"), ([2000], 8, "packed")])
@pytest.mark.parametrize("mask", [None, "causal", "prefix"])
def test_long_tiles_are_split_beside_whole_ones(lens, heads, form, mask):
    kw = {"prefix": [n // 3 for n in lens]} if mask == "prefix" else {}
    c = Case(lens, heads=heads, kv=1, form=form, tokens=max(lens) if form == "padded" else None,
             seed=41)
    out = c.run(mask=mask, **kw)
    c.check(out, mask=mask, **kw)
    again = c.run(mask=mask, **kw)  # the same bits in every run
    assert np.array_equal(out.float().cpu().numpy(), again.float().cpu().numpy())


@pytest.mark.parametrize("lens,heads,form", [
    ([1500, 200, 64, 900], 2, "packed"), ([1600, 300], 5, "padded"), ([2000], 8, "packed")])
@pytest.mark.parametrize("mask", [None, "causal", "prefix"])
@pytest.mark.parametrize("axes,cap", [(0, None), (0, 20.0), (2, None), (3, 20.0)])
def test_long_tiles_are_split_with_a_bias(lens, heads, form, mask, axes, cap):
    """The nearest keys come first within each part."""
    kw = {"prefix": [n // 3 for n in lens]} if mask == "prefix" else {}
    c = Case(lens, heads=heads, kv=1, form=form, seed=45)
    if axes:
        kw["positions"] = _places(c, axes, 3)
    c.both(mask=mask, cap=cap, slopes=np.array(SLOPES[:heads], np.float32), **kw)


@pytest.mark.parametrize("splits", [2, 4, 7])
def test_split_parts_land_in_rings_that_are_free(splits):
    """Key tiles that end with their sequence have rows of V zeroed in the ring
    that other CTAs then store parts into: many launches, one after the other,
    give the same bits, and the right ones."""
    import torch
    c = Case([449, 130, 65, 321, 700], heads=3, seed=43)
    outs = [torch.full((c.rows, 192), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(40)]
    for o in outs:
        c.run(out=o, key_splits=splits)
    for o in outs:
        assert torch.equal(o, outs[0])
    c.check(outs[0])


def test_padded_batch_without_lengths_and_strided_rows():
    import torch
    c = Case([96, 96, 96], heads=2, kv=1, form="padded", extra=3)
    out = torch.full((c.rows, 5 * 64), 7.0, device="cuda", dtype=torch.bfloat16)
    got = c.run(out=out, lengths=None, batch=3)
    c.check(got)
    assert torch.all(out[:, 128:] == 7.0)


@pytest.mark.parametrize("last,splits", [(0, 0), (0, 3), (0, 1), (2, 0), (2, 2), (100, 0)])
def test_results_in_the_places_of_q(last, splits):
    """And in columns beside the rows they come from."""
    import torch
    c = Case([300, 77, 5, 130], heads=4, kv=2, seed=51, extra=4)
    kw = dict(mask="causal", last_rows=last, key_splits=splits)
    want = c.run(**kw)
    flat = c.buf.view(torch.bfloat16).reshape(c.rows, -1)  # 8 heads of Q|K|V, 4 more
    beside = c.run(out=flat[:, 512:768], **kw)
    over = c.run(out=flat[:, :256], **kw)
    done = (want != 7.0).any(1)
    assert torch.equal(beside[done], want[done]) and torch.equal(over[done], want[done])
    assert int(done.sum()) == sum(min(last or n, n) for n in (300, 77, 5, 130))


def test_a_sequence_that_overflows_keeps_to_itself():
    """Infinite scores make their own rows NaN, as the formula does, and no others."""
    import torch
    c = Case([70, 70, 70], heads=1, seed=6)
    rows = c.qkv.view(torch.bfloat16)
    rows[70:140, :2] = 3e38
    out = c.run().float().cpu().numpy()
    assert np.isnan(out[70:140]).all()
    keep = np.r_[0:70, 140:210]
    assert np.isfinite(out[keep]).all()
    rows[70:140, :2] = 0.0
    assert np.array_equal(c.run().float().cpu().numpy()[keep], out[keep])


def test_a_dominant_score_late_in_the_sequence():
    """The running maximum grows by hundreds between tiles: the rescaling path."""
    c = Case([400], heads=1, qk="f16", seed=12)
    import torch
    for j in (100, 250, 399):
        c.qkv[j, 1] = (c.qkv[j, 0].view(torch.float16) * (1 + j / 50)).view(torch.int16)
    x = c.qkv.view(torch.float16).double().cpu().numpy()
    c.k = x[:, 1:2]
    c.both()
    c.both(mask="causal")


@pytest.mark.parametrize("slope", [None, -0.25])
def test_the_maximum_changes_hands_with_every_tile(slope):
    """Scores that rise from key tile to key tile (or, with a negative slope, away
    from the row): each of the two streams of a row's softmax takes a new
    reference from the other every time, the same bits in many launches."""
    import torch
    c = Case([1000, 260], heads=2, qk="f16", seed=47)
    kw = {"slopes": np.full(2, slope, np.float32)} if slope else {}
    if not slope:
        x = c.qkv.view(torch.float16)
        x[:, 2:4, 0] = (torch.arange(c.rows, device="cuda") / 20.0).half()[:, None]
        x[:, :2, 0] = 8.0  # a score grows by 3.2 a tile of 64 keys
        x = x.double().cpu().numpy()
        c.q, c.k = x[:, :2], x[:, 2:4]
    outs = [c.run(**kw) for _ in range(20)]
    for o in outs:
        assert torch.equal(o, outs[0])
    c.check(outs[0], **kw)


def test_offsets_and_lengths_that_point_outside_are_clamped():
    import torch
    c = Case([50, 60], heads=1, gap=0, seed=1)
    c.kw["offsets"] = torch.tensor([-4, 50, 10 ** 9], dtype=torch.int32, device="cuda")
    c.both()
    p = Case([64, 64], heads=1, form="padded")
    p.kw["lengths"] = torch.tensor([2 ** 31 - 1, 64], dtype=torch.int32, device="cuda")
    p.both()
    p.kw["lengths"] = torch.tensor([-3, 64], dtype=torch.int32, device="cuda")
    out = p.run().float().cpu().numpy()
    assert np.all(out[:64] == 7.0) and np.all(out[64:] != 7.0)


def test_expanded_tensors_are_refused():
    """Their row stride, 0, would say "side by side" and reach behind them."""
    import torch
    from beatlm_b200 import ops
    one = lambda *shape: torch.zeros(shape, device="cuda").expand(4, *shape[1:])  # noqa: E731
    x, pos, out = (torch.zeros(s, device="cuda") for s in ((4, 1, 64), (4, 2), (4, 64)))
    for args in ((one(1, 1, 64), pos), (x, one(1, 2))):
        with pytest.raises(ValueError, match="expanded"):
            ops.rope(*args, sections=(16, 16))
    with pytest.raises(ValueError, match="expanded"):
        ops.rope(x, pos, sections=(16, 16), out=one(1, 1, 64))
    qkv, slopes = torch.zeros((4, 3, 64), device="cuda").half(), torch.ones(1, device="cuda")
    for q, kw in ((one(1, 3, 64).half()[:1].expand(4, 3, 64), {}), (qkv, dict(out=one(1, 64))),
                  (qkv, dict(slopes=slopes, positions=one(1, 2)))):
        with pytest.raises(ValueError, match="expanded"):
            ops.masked_attention(q, heads=1, **{"out": out, **kw})
    # one row has no stride to speak of
    assert torch.equal(ops.rope(x[:1].expand(1, 1, 64), pos[:1], sections=(16, 16)), x[:1])


@pytest.mark.parametrize("last", [0, 1])
def test_rows_past_32_bit_offsets(last):
    """Rows 65536 values apart, the sequence behind 2^31 of them: rotation in
    place, then attention, both strided."""
    import torch
    from beatlm_b200 import ops
    rows, begin, stride = 33000, 32780, 65536
    c = Case([rows - begin], heads=2, kv=1, gap=0, seed=31)
    big = torch.empty((rows, stride), dtype=torch.int16, device="cuda")
    out = torch.empty((rows, stride), dtype=torch.bfloat16, device="cuda")
    qkv, o = big[:, :256], out[:, :128]
    qkv[begin:] = c.qkv.reshape(-1, 256)
    o.fill_(7.0)
    pos = torch.zeros((rows, 2), device="cuda")
    pos[begin:] = torch.rand((rows - begin, 2), device="cuda") * 40
    ops.rope(qkv, pos, sections=(16, 16), heads=3, head_dim=64, dtype="bf16")
    x, t = (v.reshape(-1, 4, 64)[:, :3].view(torch.bfloat16) for v in (c.qkv, qkv[begin:]))
    _check_rope(t, x.contiguous(), pos[begin:], (16, 16), "bf16", theta=100.0, pairing="half",
                inverse=False)
    offsets = torch.tensor([begin, rows], dtype=torch.int32, device="cuda")
    ops.masked_attention(qkv, heads=2, kv_heads=1, qk_dtype="bf16", offsets=offsets, mask="causal",
                         last_rows=last, out=o)
    assert torch.all(o[:begin] == 7.0)
    t = t.double().cpu().numpy()
    c.q, c.k = t[:, :2], t[:, 2:]
    c.check(o[begin:].contiguous(), mask="causal", last_rows=last)


# ------------------------------------------------------------------ as they are used

def test_a_recorded_launch_follows_its_lengths():
    """Captured once, replayed as a stream's sequences grow."""
    import torch
    c = Case([256, 256], heads=4, kv=2, form="padded", tokens=256, seed=2)
    out = torch.full((c.rows, 256), 7.0, device="cuda", dtype=torch.bfloat16)
    kw = dict(mask="causal", last_rows=1)
    c.run(out=out, **kw)  # loads what a first call loads
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(out=out, **kw)
    for lens in ([3, 200], [4, 201], [0, 256]):
        c.kw["lengths"].copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        c.where = ref.spans(2, 256, lengths=lens)
        c.check(out, **kw)


def test_two_streams_at_once():
    import torch
    cs = [Case([400, 30 + i], heads=2, seed=20 + i) for i in range(2)]
    outs = [torch.full((c.rows, 128), 7.0, device="cuda", dtype=torch.bfloat16) for c in cs]
    torch.cuda.synchronize()
    ss = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        for c, o, s in zip(cs, outs, ss):
            c.run(out=o, stream=s, mask="causal")
    torch.cuda.synchronize()
    for c, o in zip(cs, outs):
        c.check(o, mask="causal")


def _by_hand(qkv, heads, grids, sections):
    """Rotary positions and document attention of the packed rows, in 64 bits."""
    import torch
    x = qkv[:, :2 * heads].view(torch.bfloat16).double().cpu().numpy()
    off, _, pos = ref.pack(grids, qkv.shape[0], 1, False)
    turned, _ = ref.rope(x, pos[:, 1:], sections, 100.0, "axis_half", False)
    turned = torch.from_numpy(turned).to(torch.bfloat16).double().numpy()
    v = qkv[:, 2 * heads:].view(torch.float16).double().cpu().numpy()
    where = ref.spans(len(grids), qkv.shape[0], offsets=off)
    return where, turned[:, :heads], turned[:, heads:], v


@pytest.mark.parametrize("program", [False, True])
def test_pack_then_rope_then_attention(program):
    """The three in a row, as an encoder's layer uses them, by plain calls and
    as a program of prebuilt launches replayed from one graph."""
    import torch
    from beatlm_b200 import ops, runtime
    heads, grids = 2, [(1, 6, 7), (2, 3, 5), (1, 11, 13)]
    rows = sum(t * h * w + 1 for t, h, w in grids) + 5
    rng = np.random.default_rng(1)
    start = ops.pack_qkv(rng.standard_normal((rows, 3, heads, 64)), "bf16").reshape(rows, -1, 64)
    qkv = torch.empty_like(start)
    g = torch.tensor(grids, dtype=torch.int32, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    pos = torch.zeros((rows, 3), device="cuda")
    out = torch.full((rows, heads * 64), 7.0, device="cuda", dtype=torch.bfloat16)
    pk = dict(offsets=off, positions=pos, lead=1)
    rp = dict(sections=(16, 16), pairing="axis_half", heads=2 * heads, head_dim=64, dtype="bf16")
    at = dict(heads=heads, qk_dtype="bf16", offsets=off, out=out)
    flat = qkv.reshape(rows, -1)
    qkv.copy_(start)
    if program:
        k = runtime.Kernels([runtime.Spec(ops.pack_args(g, **pk), "pack"),
                             runtime.Spec(ops.rope_args(flat, pos[:, 1:], **rp), "rope"),
                             runtime.Spec(ops.masked_attention_args(qkv, **at), "attention")])
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = k.capture(s)
        graph.launch(s)
    else:
        ops.pack(g, **pk)
        ops.rope(flat, pos[:, 1:], **rp)
        ops.masked_attention(qkv, **at)
    torch.cuda.synchronize()
    where, q, kk, v = _by_hand(start, heads, grids, (16, 16))
    # Q and K against the definition; the attention on what the rotation gave
    t = qkv[:, :2 * heads].view(torch.bfloat16).double().cpu().numpy()
    both = np.concatenate([q, kk], 1)
    assert np.all(np.abs(t - both) <= np.abs(both) * 2 * ref.EPS["bf16"] + 1e-5)
    c = Case.__new__(Case)
    c.heads, c.kv, c.rows, c.where = heads, heads, rows, where
    c.q, c.k, c.v = t[:, :heads], t[:, heads:], v
    c.check(out)
