"""Refusals of the packed-batch operators: every malformed argument is turned
away on the host, before anything is launched (no GPU needed)."""
import ctypes

import numpy as np
import pytest

from beatlm_b200 import _native as N

A = 1 << 20  # an aligned address; nothing is launched, so nothing reads it


def _call(fn, a):
    N.check(fn(ctypes.byref(a), None))


def _pack(**kw):
    base = dict(images=3, capacity=100, lead=1, grids=A, offsets=2 * A, image=3 * A,
                positions=4 * A)
    base.update(kw)
    return N.PackArgs(**base)


@pytest.mark.parametrize("kw,why", [
    (dict(images=0), "no images"), (dict(capacity=0), "no rows"), (dict(grids=None), "null"),
    (dict(offsets=None), "null"), (dict(capacity=1 << 31), "32-bit"),
    (dict(lead=1 << 31), "32-bit"), (dict(images=0x7FFFFFFF), "32-bit"),
    (dict(offsets=2 * A + 2), "aligned"), (dict(positions=4 * A + 1), "aligned")])
def test_pack_refuses(kw, why):
    with pytest.raises(N.BackendError, match=why):
        _call(N.lib().bl_pack, _pack(**kw))


def _rope(sections=(16, 16), **kw):
    base = dict(rows=10, heads=4, head_dim=64, axes=2, pairing=0, dtype=N.BL_BF16, theta=100.0,
                x=A, positions=2 * A, out=A)
    base.update(kw)
    a = N.RopeArgs(**base)
    for i, n in enumerate(sections):
        a.sections[i] = n
    return a


@pytest.mark.parametrize("kw,why", [
    (dict(rows=0), "zero"), (dict(heads=0), "zero"), (dict(axes=0), "axes"),
    (dict(axes=4), "axes"), (dict(sections=(16, 0)), "no pairs"),
    (dict(sections=(16, 17)), "33 pairs"), (dict(sections=(0xFFFFFFFF, 1)), "pairs in a head"),
    (dict(sections=(100, 100), head_dim=512), "at most"), (dict(pairing=3), "pairing"),
    (dict(dtype=3), "dtype"), (dict(theta=0.0), "theta"), (dict(theta=float("inf")), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(x=None), "null"), (dict(out=None), "null"),
    (dict(positions=None), "null"), (dict(x_row_stride=255), "shorter"),
    (dict(out_row_stride=255), "shorter"), (dict(pos_row_stride=1), "shorter"),
    (dict(x=A + 1), "aligned"), (dict(positions=2 * A + 2), "aligned"),
    (dict(out_row_stride=512), "in place"), (dict(out=A + 64), "overlap"),
    (dict(out=A + 512, x_row_stride=512, out_row_stride=256), "overlap"),
    (dict(out=A + 256, x_row_stride=512, out_row_stride=512), "overlap"),
    (dict(heads=1 << 26, head_dim=64, x_row_stride=0), "values"),
    (dict(rows=1 << 31), "rows")])
def test_rope_refuses(kw, why):
    with pytest.raises(N.BackendError, match=why):
        _call(N.lib().bl_rope, _rope(**kw))


def test_rope_refuses_frequencies_that_are_not_finite():
    f = (ctypes.c_double * 32)(*([1.0] * 31 + [float("nan")]))
    with pytest.raises(N.BackendError, match="frequency 31"):
        _call(N.lib().bl_rope, _rope(freqs=ctypes.addressof(f)))


def _attn(**kw):
    base = dict(batch=2, tokens=64, heads=4, kv_heads=2, head_dim=64, scale=0.125,
                qk_dtype=N.BL_F16, v_dtype=N.BL_F16, out_dtype=N.BL_BF16, qkv=A, out=2 * A)
    base.update(kw)
    return N.MaskedAttentionArgs(**base)


@pytest.mark.parametrize("kw,why", [
    (dict(head_dim=32), "head_dim"), (dict(batch=0), "zero"), (dict(tokens=0), "zero"),
    (dict(heads=0), "zero"), (dict(kv_heads=3), "K/V heads"), (dict(heads=70000), "heads"),
    (dict(offsets=4 * A, lengths=5 * A), "packed"), (dict(batch=1 << 16, tokens=1 << 16), "rows"),
    (dict(qk_dtype=N.BL_F32), "Q/K dtype"), (dict(v_dtype=N.BL_BF16), "V dtype"),
    (dict(out_dtype=7), "out dtype"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap"),
    (dict(cap=float("nan")), "cap"), (dict(scale=0.125, cap=1e-8), "millionth"), (dict(mask=3), "mask 3"), (dict(mask=2), "prefix"),
    (dict(prefix=4 * A), "prefix"), (dict(positions=4 * A, pos_axes=2), "slopes"),
    (dict(positions=4 * A, slopes=5 * A), "position axes"),
    (dict(positions=4 * A, slopes=5 * A, pos_axes=4), "position axes"),
    (dict(positions=4 * A, slopes=5 * A, pos_axes=2, pos_row_stride=1), "shorter"),
    (dict(key_splits=9), "key splits"), (dict(qkv=None), "null"), (dict(out=None), "null"),
    (dict(qkv_row_stride=504), "stride"), (dict(qkv_row_stride=516), "stride"),
    (dict(qkv=A + 8), "alignment"), (dict(out=2 * A + 8), "alignment"),
    (dict(out_row_stride=255), "output"), (dict(out_row_stride=260), "output"),
    (dict(lengths=4 * A + 2), "4-byte")])
def test_masked_attention_refuses(kw, why):
    with pytest.raises(N.BackendError, match=why):
        _call(N.lib().bl_masked_attention, _attn(**kw))


def test_null_arguments():
    for f in ("bl_pack", "bl_rope", "bl_masked_attention"):
        with pytest.raises(N.BackendError, match="null args"):
            N.check(getattr(N.lib(), f)(None, None))


def test_programs_take_the_packed_batch_kernels():
    """Each is a kernel of its own kind that is never split; a program refuses
    what the call refuses."""
    from beatlm_b200 import runtime as R
    for a in (_pack(), _rope(), _attn()):
        assert R.max_parts(R.Spec(a, "k", parts=4)) == 1
    for a, why in ((_pack(images=0), "no images"), (_rope(pairing=9), "pairing"),
                   (_attn(mask=9), "mask 9")):
        with pytest.raises(N.BackendError, match=why):
            R.Kernels([R.Spec(a, "k")])


def test_python_calls_refuse_cpu_tensors():
    import torch
    from beatlm_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.pack(torch.ones((2, 3), dtype=torch.int32), offsets=torch.zeros(3, dtype=torch.int32),
                 capacity=4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope(torch.zeros((2, 1, 64)), torch.zeros((2, 2)), sections=(16, 16))
    with pytest.raises(ValueError, match="CUDA"):
        ops.masked_attention(torch.zeros((2, 3, 64), dtype=torch.int16), heads=1,
                             out=torch.zeros((2, 64)))


@pytest.fixture
def on_cpu(monkeypatch):
    """The calls' own checks, without a GPU: argument structs are made of CPU
    tensors and nothing is launched."""
    from beatlm_b200 import ops
    monkeypatch.setattr(ops, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(ops, "_launch", lambda *a: pytest.fail("launched"))
    return ops


@pytest.mark.parametrize("container,out_dtype", [
    ("int16", "f32"), ("float16", "f32"), ("bfloat16", "f32"), ("float16", "bf16"),
    ("bfloat16", "f16"), ("float32", "f16"), ("int32", "bf16"), ("uint8", "f16"),
    ("float64", "f32"), ("float64", None), ("int16", None), ("int32", None)])
def test_an_output_of_another_type_or_size_is_refused(on_cpu, container, out_dtype):
    """Four-byte results in two-byte rows would end behind the buffer."""
    import torch
    qkv = torch.zeros((5, 3, 64), dtype=torch.int16)
    out = torch.zeros((5, 64), dtype=getattr(torch, container))
    for call in (on_cpu.masked_attention_args, on_cpu.masked_attention):
        with pytest.raises(ValueError, match="masked attention: .* results in an out of"):
            call(qkv, heads=1, out=out, out_dtype=out_dtype)


@pytest.mark.parametrize("container,out_dtype,code", [
    ("float32", None, N.BL_F32), ("float16", None, N.BL_F16), ("bfloat16", "bf16", N.BL_BF16),
    ("int16", "f16", N.BL_F16), ("int16", "bf16", N.BL_BF16), ("int32", "f32", N.BL_F32)])
def test_outputs_and_containers_that_fit(on_cpu, container, out_dtype, code):
    import torch
    a = on_cpu.masked_attention_args(torch.zeros((5, 3, 64), dtype=torch.int16), heads=1,
                                     out=torch.zeros((5, 64), dtype=getattr(torch, container)),
                                     out_dtype=out_dtype)
    assert a.out_dtype == code


# 128 rows of 512 values of Q|K|V (1024 bytes), 256 values of output (512 bytes in 16 bits)
@pytest.mark.parametrize("kw", [
    dict(out=A + 512, out_row_stride=512), dict(out=A + 768, out_row_stride=512), dict(out=A),
    dict(out=A, out_row_stride=512, out_dtype=N.BL_F32), dict(out=A + 127 * 1024 + 1008),
    dict(out=A - 127 * 512), dict(out=A, qkv_row_stride=768, out_row_stride=512),
    dict(out=A + 1008, qkv_row_stride=768, out_row_stride=768),
    dict(out=A + 1040, qkv_row_stride=768, out_row_stride=768),
    dict(out=A - 496, qkv_row_stride=768, out_row_stride=768),
    dict(out=A + 1024, qkv_row_stride=768, out_row_stride=384, out_dtype=N.BL_F32),
    dict(out=A + 16, batch=1, tokens=1), dict(out=A, batch=1, tokens=1, out_dtype=N.BL_F32)])
def test_an_output_over_rows_still_read_is_refused(kw):
    with pytest.raises(N.BackendError, match="out overlaps qkv"):
        _call(N.lib().bl_masked_attention, _attn(**kw))


@pytest.mark.parametrize("kw", [
    dict(out=A, out_row_stride=512), dict(out=A, batch=1, tokens=1),
    dict(out=A + 128 * 1024), dict(out=A - 128 * 512),
    dict(out=A + 1024, qkv_row_stride=768, out_row_stride=768),
    dict(out=A - 512, qkv_row_stride=768, out_row_stride=768)])
def test_outputs_apart_and_over_q_pass_the_overlap_check(kw):
    """(No GPU here: what comes after the check of arguments fails, otherwise.)"""
    with pytest.raises(N.BackendError, match="4-byte"):
        _call(N.lib().bl_masked_attention, _attn(lengths=4 * A + 2, **kw))


@pytest.mark.parametrize("tensor,qk_dtype", [
    ("bfloat16", "f16"), ("bfloat16", "bf16"), ("float16", "bf16")])
def test_rows_of_another_type_than_they_are_read_as_are_refused(on_cpu, tensor, qk_dtype):
    """A bfloat16 tensor's V is not f16, whatever its Q and K are read as."""
    import torch
    out = torch.zeros((5, 64), dtype=torch.float16)
    for shape in ((5, 3, 64), (5, 192)):
        qkv = torch.zeros(shape, dtype=getattr(torch, tensor))
        for call in (on_cpu.masked_attention_args, on_cpu.masked_attention):
            with pytest.raises(ValueError, match="beside f16 V in a tensor of torch." + tensor):
                call(qkv, heads=1, out=out, qk_dtype=qk_dtype)
    for t, qk in ((torch.float16, "f16"), (torch.int16, "f16"), (torch.int16, "bf16")):
        on_cpu.masked_attention_args(torch.zeros((5, 192), dtype=t), heads=1, out=out, qk_dtype=qk)


def _encoder(**kw):
    from beatlm_b200 import model as M
    cfg = M.ViTConfig(dim=128, heads=2, mlp=256, layers=0, patch=4, side=8, cin=3, out_indices=())
    n = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    w = {"blocks": [], "patch_w": n(cfg.taps, 128), "patch_b": n(128), "norm_g": n(128),
         "norm_b": n(128)}
    return cfg, M.PackedEncoder(cfg, w, capacity=50, images=4, dtype="f16", device="cpu", **kw)


@pytest.mark.parametrize("mask", ["prefix", "document", 1])
def test_the_packed_encoder_refuses_masks_it_has_no_way_to_run(mask):
    """A prefix mask needs lengths, which the encoder does not take."""
    with pytest.raises(ValueError, match="mask"):
        _encoder(mask=mask)
    for m in (None, "none", "causal"):
        _encoder(mask=m)


def test_the_packed_encoder_refuses_sizes_and_patches_of_other_forms():
    """Sizes of one column would be spread over (t, h, w), bits in an integer
    container taken for numbers."""
    import torch
    cfg, enc = _encoder()
    rows, sizes = torch.zeros((6, cfg.k_pad), dtype=torch.float16), torch.ones((2, 3), dtype=torch.int32)
    for r, g in ((rows, sizes[:, :1]), (rows, sizes[0]), (rows, torch.ones((2, 2, 3))),
                 (rows.view(torch.int16), sizes), (rows[None], sizes), (rows[:, :5], sizes),
                 (rows[0], sizes)):
        with pytest.raises(ValueError, match="images with"):
            enc.forward(r, g)


@pytest.mark.parametrize("container,out_dtype", [
    ("int16", "f32"), ("float16", "f32"), ("uint8", "f16"), ("float32", "bf16")])
def test_the_dense_attention_refuses_outputs_of_another_size(container, out_dtype):
    import torch
    from beatlm_b200 import ops
    qkv = torch.zeros((1, 5, 3, 1, 64), dtype=torch.int16)
    out = torch.zeros((1, 5, 64), dtype=getattr(torch, container))
    with pytest.raises(ValueError, match="attention: .* results in an out of"):
        ops.attention_args(qkv, tokens=5, heads=1, out=out, out_dtype=out_dtype)
    for fits, name in ((torch.int16, "bf16"), (torch.float16, None), (torch.float32, "f32")):
        ops.attention_args(qkv, tokens=5, heads=1, out=torch.zeros((1, 5, 64), dtype=fits),
                           out_dtype=name)


@pytest.mark.parametrize("kw", [
    dict(scale=1e4, cap=0.0101),  # scale (scale / cap)^6, the last coefficient of the series
    dict(scale=1.0, cap=3e38), dict(scale=3e38), dict(scale=3e38, cap=1e36)])
def test_scores_whose_constants_leave_32_bits_are_refused(kw):
    """An infinite constant times a score of zero is NaN."""
    with pytest.raises(N.BackendError, match="32 bits"):
        _call(N.lib().bl_masked_attention, _attn(**kw))
    with pytest.raises(N.BackendError, match="4-byte"):  # well within them
        _call(N.lib().bl_masked_attention, _attn(scale=1e3, cap=0.00101, lengths=4 * A + 2))
