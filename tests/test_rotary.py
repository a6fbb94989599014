"""Rotation, rotated append and block scales without a GPU: plans against their
formulas, and what the C ABI and the Python checks refuse before they touch a
device."""
import ctypes
import math

import pytest
import torch

import rotary_oracle as RO
from test_paged import record

P = ctypes.c_void_p(0x100000)
A = 0x100000

SCALINGS = [
    None, {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "ntk", "factor": 3.0},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 32768},
    {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 500, "beta_slow": 2, "beta_fast": 20},
    {"rope_type": "wavelength", "factor": 8.0, "original_max_position_embeddings": 8192},
    {"rope_type": "wavelength", "factor": 2.0, "original_max_position_embeddings": 4096, "low_freq_factor": 0.5, "high_freq_factor": 9},
]


@pytest.mark.parametrize("rotary,theta", [(2, 10000.0), (20, 10000.0), (64, 10000000.0), (128, 500000.0)])
@pytest.mark.parametrize("scaling", SCALINGS, ids=str)
def test_plan_frequencies(fp8lin, scaling, rotary, theta):
    plan = fp8lin.rotary_plan(rotary, theta, scaling, device="cpu")
    freq, magnitude = RO.frequencies(rotary, theta, scaling)
    assert plan.steps.dtype == torch.int64 and plan.steps.shape == (rotary // 2,) and not plan.neighbours
    assert math.isclose(plan.magnitude, magnitude, rel_tol=1e-15)
    for got, f in zip(plan.steps.tolist(), freq):
        got = (got % 2 ** 64) / 2 ** 64
        assert got * 2 ** 64 % 4 == 0
        # powers in 64 bits, a few half steps off each: of a turn per position
        assert math.isclose(got, f / (2 * math.pi), rel_tol=64 * 2 ** -53, abs_tol=2 ** -62)


def test_plan_of_frequencies_and_sections(fp8lin):
    freq = [1.0, 0.25, 1e-9, 7.0, -0.5, 0.0]
    plan = fp8lin.rotary_plan(12, frequencies=freq, magnitude=1.5, neighbours=True, sections=[2, 1, 2], device="cpu")
    axes = [0, 1, 2, 0, 0, 2]
    assert [s % 2 ** 64 for s in plan.steps.tolist()] == RO.steps(freq, axes)
    assert plan.magnitude == 1.5 and plan.neighbours
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 100, "attention_factor": 1.25}
    assert fp8lin.rotary_plan(8, 1e4, yarn, device="cpu").magnitude == 1.25
    # a whole turn a position turns nothing
    assert fp8lin.rotary_plan(2, frequencies=[2 * math.pi], device="cpu").steps.tolist() == [0]


@pytest.mark.parametrize("args,kw", [
    ((0,), {}), ((7,), {}), ((-2,), {}), ((8,), dict(theta=0.0)), ((8,), dict(theta=math.inf)), ((8,), dict(theta=-5.0)),
    ((8,), dict(scaling={"rope_type": "dynamic", "factor": 2.0})), ((8,), dict(scaling={"rope_type": "linear", "factor": 0.0})),
    ((8,), dict(scaling={"rope_type": "linear", "factor": math.nan})), ((8,), dict(scaling={"rope_type": "yarn", "factor": 2.0})),
    ((8,), dict(scaling={"rope_type": "wavelength", "factor": 2.0, "original_max_position_embeddings": 100, "low_freq_factor": 4})),
    ((8,), dict(theta=1.0, scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 100})),
    ((8,), dict(frequencies=[1.0])), ((4,), dict(frequencies=[1.0, math.inf])), ((4,), dict(frequencies=[1.0, 2.0], scaling={"rope_type": "linear"})),
    ((8,), dict(sections=[1, 2])),
], ids=str)
def test_plan_refusals(fp8lin, args, kw):
    with pytest.raises(fp8lin.Fp8linError):
        fp8lin.rotary_plan(*args, device="cpu", **kw)


def test_steps_validation(fp8lin):
    L = fp8lin.lib()
    f, axes, out = (ctypes.c_double * 2)(1.0, 2.0), (ctypes.c_int32 * 2)(0, 4), (ctypes.c_uint64 * 2)()
    assert L.fp8lin_rotary_steps(f, None, 2, out) == 0 and L.fp8lin_rotary_steps(None, None, 0, None) == 0
    assert L.fp8lin_rotary_steps(f, axes, 2, out) == 2 and L.fp8lin_rotary_steps(None, None, 2, out) == 2
    assert L.fp8lin_rotary_steps(f, None, 2, None) == 2 and L.fp8lin_rotary_steps(f, None, -1, out) == 1
    mag = ctypes.c_double()
    call = L.fp8lin_rotary_frequencies
    assert call(4, 1e4, 0, 1.0, 0.0, 0.0, 0.0, f, ctypes.byref(mag)) == 0
    assert call(4, 1e4, 5, 1.0, 0.0, 0.0, 0.0, f, ctypes.byref(mag)) == 2 and call(4, 1e4, 0, 1.0, 0.0, 0.0, 0.0, None, ctypes.byref(mag)) == 2
    assert call(3, 1e4, 0, 1.0, 0.0, 0.0, 0.0, f, ctypes.byref(mag)) == 1


def rotary(fp8lin, **kw):
    from fp8lin._lib import RotaryRecord
    return RotaryRecord(**{**dict(steps=A + 0x900000, rotary=32, neighbours=0, magnitude=1.0), **kw})


def rotate(fp8lin, plan=None, null=False, **kw):
    d = dict(x=A, x_token=256, x_head=64, tokens=5, heads=4, head_dim=64, positions=A + 0x800000, axes=1, axis_stride=0, transposed=0,
             y=A + 0x400000, y_token=256, y_head=64, stream=None)
    d.update(kw)
    rec = plan if plan is not None else rotary(fp8lin)
    return fp8lin.lib().fp8lin_rotate(None if null else ctypes.byref(rec), *d.values())


# a call that passes the checks ends at the device: there is none here (6), or the launch is refused on a GPU box
@pytest.mark.parametrize("change,code", [
    (dict(null=True), 2), (dict(x=None), 2), (dict(y=None), 2), (dict(positions=None), 2), (dict(tokens=-1), 1), (dict(heads=-1), 1),
    (dict(head_dim=63), 1), (dict(head_dim=0), 1), (dict(head_dim=1026), 1), (dict(axes=0), 1), (dict(axes=5), 1), (dict(axis_stride=-1), 1),
    (dict(x_token=-256), 1), (dict(y_head=1 << 60), 1), (dict(tokens=1 << 30), 1), (dict(tokens=0), 0), (dict(heads=0), 0),
    (dict(y=A + 2), 2), (dict(y=A + 64 * 2), 2), (dict(y=A, y_token=512), 2), (dict(positions=A + 0x400000), 2), (dict(y_token=128), 2),
    (dict(heads=1 << 30, tokens=1), 1), (dict(y_head=32), 2), (dict(y_token=0), 2), (dict(y_token=64, y_head=64), 2), (dict(y=A + 0x900000), 2),
], ids=str)
def test_rotate_validation(fp8lin, change, code):
    assert rotate(fp8lin, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(steps=None), 2), (dict(steps=A + 4), 2), (dict(rotary=0), 1), (dict(rotary=31), 1), (dict(rotary=66), 1), (dict(magnitude=math.nan), 2),
    (dict(magnitude=math.inf), 2),
], ids=str)
def test_rotate_plan_validation(fp8lin, change, code):
    assert rotate(fp8lin, plan=rotary(fp8lin, **change)) == code


def blocks(**kw):
    from fp8lin._lib import BlockScalesRecord
    return BlockScalesRecord(**{**dict(k=A + 0x700000, v=A + 0x701000, block=16), **kw})


def cache8(fp8lin, **kw):
    return record(fp8lin, **{**dict(k=A + 0x500000, v=A + 0x600000, fp8=1), **kw})


def append(fp8lin, rec=None, scales=None, plan=None, **kw):
    d = dict(q=A, q_token=256, q_head=64, heads=4, k=A + 0x100000, k_token=128, k_head=64, v=A + 0x200000, v_token=128, v_head=64,
             q_norm=A + 0x300000, k_norm=A + 0x301000, eps=1e-6, centered=1, positions=A + 0x800000, axes=1, axis_stride=0, slots=A + 0x810000,
             tokens=5, q_out=A + 0x400000, out_token=256, out_head=64, stream=None)
    d.update(kw)
    return fp8lin.lib().fp8lin_paged_rotate_append(
        None if rec is False else ctypes.byref(rec if rec is not None else cache8(fp8lin)),
        None if scales is False else ctypes.byref(scales if scales is not None else blocks()),
        None if plan is False else ctypes.byref(plan if plan is not None else rotary(fp8lin)), *d.values())


@pytest.mark.parametrize("change,code", [
    (dict(rec=False), 2), (dict(q=None), 2), (dict(q_out=None), 2), (dict(k=None), 2), (dict(v=None), 2), (dict(slots=None), 2),
    (dict(positions=None), 2), (dict(tokens=-1), 1), (dict(heads=-1), 1), (dict(tokens=1 << 30), 1), (dict(eps=-1.0), 2), (dict(eps=math.nan), 2),
    (dict(eps=math.inf), 2), (dict(axes=7), 1), (dict(k_token=-1), 1), (dict(tokens=0, q=None, k=None), 0), (dict(scales=False), 2),
    (dict(q_out=A + 64), 2), (dict(q_out=A + 0x100000), 2), (dict(q_out=A + 0x500000), 2), (dict(q_out=A + 0x700000), 2), (dict(out_token=128), 2),
    (dict(k=A + 0x500000), 2), (dict(slots=A + 0x600000), 2), (dict(positions=A + 0x700000), 2), (dict(k_norm=A + 0x400000), 2),
    (dict(q_out=A, out_token=512, q_token=256), 2),
], ids=str)
def test_append_validation(fp8lin, change, code):
    assert append(fp8lin, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(k=None), 2), (dict(v=0), 2), (dict(block=8), 1), (dict(block=0), 1), (dict(block=32), 1), (dict(block=24), 1), (dict(block=-16), 1),
    (dict(k=A + 0x500000), 2), (dict(k=A + 0x701000), 2),
], ids=str)
def test_block_scales_validation(fp8lin, change, code):
    assert append(fp8lin, scales=blocks(**change)) == code


def test_append_caches(fp8lin):
    # block scales need an 8-bit cache without other scales
    assert append(fp8lin, rec=cache8(fp8lin, fp8=0)) == 2
    assert append(fp8lin, rec=cache8(fp8lin, k_scale=0x100, v_scale=0x200)) == 2
    wide = dict(k_slot=4096, v_slot=4096, k_page=65536, v_page=65536)
    assert append(fp8lin, rec=cache8(fp8lin, head_dim=56, **wide)) == 3
    assert append(fp8lin, rec=cache8(fp8lin, head_dim=2048, **wide)) == 3
    assert append(fp8lin, rec=cache8(fp8lin, page_size=512, **wide), scales=blocks(block=256)) == 1
    assert append(fp8lin, rec=cache8(fp8lin, k_page=1 << 60)) == 1


def test_python_refuses_host_tensors(fp8lin):
    plan = fp8lin.rotary_plan(32, device="cpu")
    x = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    at = torch.zeros(5, dtype=torch.int64)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.uint8)
    scale = torch.zeros(4, 1, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    for call in (lambda: fp8lin.rotate(x, at, plan),
                 lambda: fp8lin.paged_rotate_append(x, x, x, at, at, cache, cache, plan, k_scale=scale, v_scale=scale),
                 lambda: fp8lin.paged_append(x, x, at, cache, cache, k_scale=scale, v_scale=scale)):
        with pytest.raises(fp8lin.Fp8linError):
            call()


@pytest.mark.parametrize("change,code", [
    # a token's row of 1024: queries of 64 in each 128 of its first 448, keys from 512 on, values from 640 on; 5 tokens
    (dict(), 0), (dict(k=A + 2 * 447), 2), (dict(k=A + 2 * 448), 0), (dict(k=A + 2 * 896), 0), (dict(k=A + 2 * 897), 2),
    (dict(k=A + 2 * (4 * 1024 + 447)), 2), (dict(k=A + 2 * (4 * 1024 + 448)), 0), (dict(v=A - 2 * (4 * 1024 + 127)), 2),
    (dict(v=A - 2 * (4 * 1024 + 128)), 0),
], ids=str)
def test_append_in_place_in_one_matrix(fp8lin, change, code):
    """Queries turned in place in the projection's rows, beside the keys and values."""
    if not code and torch.cuda.is_available():
        pytest.skip("what passes the checks would be launched on these addresses")
    d = dict(q=A, q_token=1024, q_head=128, q_out=A, out_token=1024, out_head=128, k=A + 2 * 512, k_token=1024, v=A + 2 * 640, v_token=1024,
             q_norm=A + 0x300000, k_norm=A + 0x301000)
    # without a GPU what passes ends at the device
    assert append(fp8lin, **{**d, **change}) == (code or 6)


def test_the_oracle_by_differences():
    """The transposed rotation is the gradient of the rotation, by differences."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(2, 1, 8, generator=g, dtype=torch.float64), torch.randn(2, 1, 8, generator=g, dtype=torch.float64)
    at, freq = torch.tensor([3, 70001]), [1.0, 0.3, 0.01]
    for nb in (False, True):
        grad = RO.rotate(w, at, freq, 1.3, nb, transposed=True)[0]
        for i in range(16):
            d = torch.zeros(16, dtype=torch.float64)
            d[i] = 1e-3
            up, down = [(RO.rotate(x + e * d.view(x.shape), at, freq, 1.3, nb)[0] * w).sum() for e in (1, -1)]
            # the rotation is linear: differences are exact but for their own roundings
            assert abs(float((up - down) / 2e-3 - grad.flatten()[i])) < 1e-10


def test_the_oracle_of_blocks():
    """A block that grows, one that starts anew, and one that neither does, by hand."""
    assert [RO.power(v) for v in (0.0, 448.0, 448.1, 896.0, 1.75, 1.76, 2.0 ** -111)] == [-120, 0, 1, 1, -8, -7, -119]
    cache = torch.full((3, 16, 1, 16), 2.0).to(torch.float8_e4m3fn)
    powers = torch.full((3, 1, 1), 127, dtype=torch.uint8)
    rows = torch.zeros(3, 1, 16, dtype=torch.float64)
    rows[0, 0, 0], rows[1, 0, 3], rows[2, 0, 5] = 900.0, -1.75, 3.0
    values, _, bytes_, other = RO.append_blocks(rows, torch.zeros_like(rows), [17, 0, 33], cache, powers, 16)
    assert bytes_.flatten().tolist() == [119, 129, 127] == other.flatten().tolist()
    assert float(values[1, 1, 0, 0]) == 225.0 and float(values[1, 2, 0, 0]) == 0.5
    assert float(values[0, 0, 0, 3]) == -448.0 and float(values[0, 1, 0, 0]) == 2.0
    assert float(values[2, 1, 0, 5]) == 3.0 and float(values[2, 0, 0, 0]) == 2.0
