"""The encoder over a packed batch (row maps, rotary positions, attention by
image, prebuilt as one program) against the block's formulas in 64 bits."""
import numpy as np
import pytest

import packed_reference as ref

pytestmark = pytest.mark.gpu

# Every operand of a product, every output of one that feeds another, the
# rotated Q and K and the probabilities are rounded to f16, about ten roundings
# a block of at most 2^-11 of a value each; at worst they add up.
ROUNDINGS, STEP = 10, 2.0 ** -11


def _cfg(layers=2):
    from beatlm_b200.model import ViTConfig
    return ViTConfig(dim=128, heads=2, mlp=256, layers=layers, patch=4, side=8, cin=3,
                     out_indices=())


def _weights(cfg, seed):
    from beatlm_b200 import model as M
    rng = np.random.default_rng(seed)
    blocks = []
    for i in range(cfg.layers):
        w = M.block_weights_normal(rng, cfg.dim, cfg.mlp, std=cfg.dim ** -0.5)
        blocks.append(w)
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)
    return {"blocks": blocks, "patch_w": n(cfg.taps, cfg.dim) * cfg.taps ** -0.5,
            "patch_b": n(cfg.dim) * 0.1, "norm_g": 1 + 0.1 * n(cfg.dim), "norm_b": 0.1 * n(cfg.dim)}


def _f16(x):
    return np.asarray(x, np.float32).astype(np.float16).astype(np.float64)


def _ln(x, g, b, eps):
    d = x - x.mean(1, keepdims=True)
    return d / np.sqrt((d * d).mean(1, keepdims=True) + eps) * g + b


def _reference(cfg, weights, patches, grids, sections, **attn):
    from scipy.special import erf
    off, _, pos = ref.pack(grids, patches.shape[0], 0, False)
    where = ref.spans(len(grids), patches.shape[0], offsets=off)
    x = _f16(patches) @ _f16(weights["patch_w"]) + weights["patch_b"]
    if attn.get("slopes") is not None:
        attn["positions"] = pos
    for w in weights["blocks"]:
        shape = lambda k, a, b: _f16(w[k]).reshape(a, b)
        d, m, h = cfg.dim, cfg.mlp, cfg.heads
        qkv = _ln(x, w["norm1_g"], w["norm1_b"], cfg.eps) @ shape("qkv_w", d, 3 * d) + w["qkv_b"]
        q, k, v = (qkv[:, i * d:(i + 1) * d].reshape(-1, h, 64) for i in range(3))
        turn = lambda t: ref.rope(t, pos[:, 3 - len(sections):], sections, 100.0, "axis_half", False)[0]
        o, _, _ = ref.attention(turn(q), turn(k), v, where, **attn)
        x = x + w["ls1"] * (o.reshape(-1, d) @ shape("proj_w", d, d) + w["proj_b"])
        hid = _ln(x, w["norm2_g"], w["norm2_b"], cfg.eps) @ shape("fc1_w", d, m) + w["fc1_b"]
        hid = 0.5 * hid * (1 + erf(hid / np.sqrt(2)))
        x = x + w["ls2"] * (hid @ shape("fc2_w", m, d) + w["fc2_b"])
    return _ln(x, weights["norm_g"], weights["norm_b"], cfg.eps), off


def _patches(cfg, rows, seed):
    x = np.zeros((rows, cfg.k_pad), np.float32)
    x[:, :cfg.taps] = np.random.default_rng(seed).standard_normal((rows, cfg.taps))
    return x


@pytest.mark.parametrize("kw", [
    dict(), dict(sections=(12, 10, 10)), dict(cap=20.0, slopes=[0.1, 0.02]), dict(mask="causal")])
def test_packed_encoder_matches_the_formulas(kw):
    import torch
    from beatlm_b200 import model as M
    cfg = _cfg()
    w = _weights(cfg, 3)
    grids = [(1, 9, 11), (2, 4, 6), (1, 1, 1), (1, 13, 10)]
    rows = sum(t * a * b for t, a, b in grids)
    enc = M.PackedEncoder(cfg, w, capacity=rows + 40, images=6, dtype="f16", **kw)
    x = _patches(cfg, rows, 5)
    got = enc.forward(torch.from_numpy(x).half().cuda(),
                      torch.tensor(grids, dtype=torch.int32).cuda())[:rows].double().cpu().numpy()
    attn = {k: v for k, v in kw.items() if k != "sections"}
    want, off = _reference(cfg, w, x[:, :cfg.taps], grids, kw.get("sections", (16, 16)), **attn)
    assert enc.offsets.tolist() == list(off) + [rows, rows]
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= cfg.layers * ROUNDINGS * STEP, rel


def test_one_graph_runs_batches_of_other_sizes():
    """Sizes are device data: the recorded program follows them, and an image
    gives the same rows whatever shares its batch."""
    import torch
    from beatlm_b200 import model as M
    cfg = _cfg()
    enc = M.PackedEncoder(cfg, _weights(cfg, 4), capacity=400, images=5, dtype="f16")
    s = torch.cuda.Stream()
    graph = enc.program().capture(s)
    rng = np.random.default_rng(8)
    x = _patches(cfg, 150, 9)
    alone = None
    for grids in ([(1, 10, 15)], [(1, 7, 7), (1, 10, 15), (3, 5, 5)], [(1, 2, 9), (1, 10, 15)]):
        at = grids.index((1, 10, 15))
        before = sum(t * a * b for t, a, b in grids[:at])
        total = sum(t * a * b for t, a, b in grids)
        p = _patches(cfg, total, int(rng.integers(1000)))
        p[before:before + 150] = x
        with torch.cuda.stream(s):
            enc.grids.zero_()
            enc.grids[:len(grids)].copy_(torch.tensor(grids, dtype=torch.int32))
            enc.patches[:total].copy_(torch.from_numpy(p).half())
            graph.launch(s)
        s.synchronize()
        got = enc.out[before:before + 150].double().cpu().numpy()
        if alone is None:
            alone = got
        rel = np.linalg.norm(got - alone) / np.linalg.norm(alone)
        assert rel <= cfg.layers * ROUNDINGS * STEP, (grids, rel)


def test_packed_encoder_refuses_what_does_not_fit():
    import torch
    from beatlm_b200 import model as M
    cfg = _cfg(1)
    enc = M.PackedEncoder(cfg, _weights(cfg, 4), capacity=100, images=2, dtype="f16")
    grids = torch.ones((3, 3), dtype=torch.int32, device="cuda")
    rows = torch.zeros((3, cfg.k_pad), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="3 images"):
        enc.forward(rows, grids)
    with pytest.raises(ValueError, match="patch rows"):
        enc.forward(torch.zeros((101, cfg.k_pad), dtype=torch.float16, device="cuda"), grids[:2])
    with pytest.raises(ValueError, match="heads of 64"):
        M.PackedEncoder(M.ViTConfig(dim=128, heads=4, layers=0), {"blocks": []}, 10, 1)


@pytest.mark.parametrize("t,h", [(1370, 6), (300, 3)])
def test_without_masks_it_is_the_dense_attention(t, h):
    """One whole sequence: the same function as ``ops.attention``, whose stated
    tolerance each of the two may be off by (relative L2 1e-3 each)."""
    import torch
    import beatlm_b200 as bl
    from beatlm_b200 import ops
    x = np.random.default_rng(t).standard_normal((1, t, 3, h, 64)).astype(np.float32)
    qkv = bl.pack_qkv(x, "bf16")
    want = bl.attention(qkv, tokens=t, heads=h, qk_dtype="bf16")[0].double()
    got = ops.masked_attention(qkv.reshape(t, 3 * h, 64), heads=h, qk_dtype="bf16",
                               out_dtype="f32").double()
    assert float((got - want).norm() / want.norm()) <= 2e-3


def test_rows_that_were_not_given_are_zeros_and_recorded():
    """Grids that ask for more patch rows than a call gives: what is missing is
    zeros, never the rows of the batch before, and the status word says so."""
    import torch
    import beatlm_b200 as bl
    from beatlm_b200 import model as M
    cfg = _cfg()
    w = _weights(cfg, 6)
    enc = M.PackedEncoder(cfg, w, capacity=260, images=3, dtype="f16")
    dev = lambda x: torch.from_numpy(x).half().cuda()  # noqa: E731
    sizes = lambda g: torch.tensor(g, dtype=torch.int32, device="cuda")  # noqa: E731
    enc.forward(dev(_patches(cfg, 250, 12)), sizes([(1, 10, 25)]))
    torch.cuda.synchronize()
    assert bl.status(reset=True).code == 0
    grids, given = [(1, 8, 9), (1, 11, 12)], 100
    x = _patches(cfg, 72 + 132, 13)
    x[given:] = 0.0
    got = enc.forward(dev(x[:given]), sizes(grids))[:204].double().cpu().numpy()
    assert bl.status(reset=True).code == 0x50
    want, _ = _reference(cfg, w, x[:, :cfg.taps], grids, (16, 16))
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= cfg.layers * ROUNDINGS * STEP, rel
    enc.forward(dev(x[:204]), sizes(grids))
    torch.cuda.synchronize()
    assert bl.status(reset=True).code == 0


def _formulas(cfg, weights, patches, grids, dtype="f16", sections=(16, 16), pairing="axis_half",
              normalized=False, **attn):
    """_reference for every option, operands rounded as `dtype` holds them."""
    from scipy.special import erf
    from beatlm_b200.model import _round
    held = lambda a: np.asarray(_round(np.asarray(a, np.float32), dtype), np.float64)  # noqa: E731
    off, _, pos = ref.pack(grids, patches.shape[0], 0, normalized)
    where = ref.spans(len(grids), patches.shape[0], offsets=off)
    x = held(patches) @ held(weights["patch_w"]) + weights["patch_b"]
    if attn.get("slopes") is not None:
        attn["positions"] = pos
    d, m, h = cfg.dim, cfg.mlp, cfg.heads
    turn = lambda t: ref.rope(t, pos[:, 3 - len(sections):], sections, 100.0, pairing, False)[0]  # noqa: E731
    for w in weights["blocks"]:
        mat = lambda k, a, b: held(w[k]).reshape(a, b)  # noqa: E731
        qkv = _ln(x, w["norm1_g"], w["norm1_b"], cfg.eps) @ mat("qkv_w", d, 3 * d) + w["qkv_b"]
        q, k, v = (qkv[:, i * d:(i + 1) * d].reshape(-1, h, 64) for i in range(3))
        o, _, _ = ref.attention(turn(q), turn(k), v, where, **attn)
        x = x + w["ls1"] * (o.reshape(-1, d) @ mat("proj_w", d, d) + w["proj_b"])
        hid = _ln(x, w["norm2_g"], w["norm2_b"], cfg.eps) @ mat("fc1_w", d, m) + w["fc1_b"]
        hid = 0.5 * hid * (1 + erf(hid / np.sqrt(2)))
        x = x + w["ls2"] * (hid @ mat("fc2_w", m, d) + w["fc2_b"])
    return _ln(x, weights["norm_g"], weights["norm_b"], cfg.eps)


# options, and what each of them is without: the formulas then give something else
@pytest.mark.parametrize("kw,others", [
    (dict(cap=1.0, slopes=[0.5, 0.2]), [dict(cap=None), dict(slopes=None), dict(slopes=[0.5, 0.0]),
                                        dict(mask="causal")]),
    (dict(cap=1.0, slopes=[0.5, 0.2], mask="causal"), [dict(cap=None), dict(slopes=[0.0, 0.2]),
                                                       dict(mask=None)]),
    (dict(normalized=True), [dict(normalized=False)]),
    (dict(pairing="half"), [dict(pairing="axis_half")]),
    (dict(pairing="adjacent", sections=(8, 12, 12)), [dict(pairing="axis_half"),
                                                      dict(sections=(12, 10, 10))])])
def test_packed_encoder_options_are_there(kw, others):
    import torch
    from beatlm_b200 import model as M
    cfg = _cfg()
    w = _weights(cfg, 3)
    grids = [(1, 9, 11), (2, 4, 6), (1, 1, 1), (1, 13, 10)]
    rows = sum(t * a * b for t, a, b in grids)
    x = _patches(cfg, rows, 5)
    want = _formulas(cfg, w, x[:, :cfg.taps], grids, **kw)
    far = lambda a: np.linalg.norm(a - want) / np.linalg.norm(want)  # noqa: E731
    most = cfg.layers * ROUNDINGS * STEP
    for other in others:
        assert far(_formulas(cfg, w, x[:, :cfg.taps], grids, **{**kw, **other})) > 3 * most, other
    enc = M.PackedEncoder(cfg, w, capacity=rows + 3, images=4, dtype="f16", **kw)
    got = enc.forward(torch.from_numpy(x).half().cuda(),
                      torch.tensor(grids, dtype=torch.int32).cuda())[:rows].double().cpu().numpy()
    assert far(got) <= most, far(got)


@pytest.mark.parametrize("kw", [dict(), dict(cap=1.0, slopes=[0.5, 0.2])])
def test_packed_encoder_in_bf16(kw):
    """The default type: bf16 Q and K beside f16 V, steps of 2^-8."""
    import torch
    from beatlm_b200 import model as M
    cfg = _cfg()
    w = _weights(cfg, 7)
    grids = [(1, 9, 11), (1, 14, 10), (3, 5, 2)]
    rows = sum(t * a * b for t, a, b in grids)
    x = _patches(cfg, rows, 5)
    want = _formulas(cfg, w, x[:, :cfg.taps], grids, dtype="bf16", **kw)
    enc = M.PackedEncoder(cfg, w, capacity=rows, images=3, **kw)
    got = enc.forward(torch.from_numpy(x).bfloat16().cuda(),
                      torch.tensor(grids, dtype=torch.int32).cuda())[:rows].double().cpu().numpy()
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= cfg.layers * ROUNDINGS * 2.0 ** -8, rel
