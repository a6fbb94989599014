"""A model config's dict in rotary_plan: every key is read or refused, and none
that changes the rotation is left aside (no GPU)."""
import math

import pytest

import rotary_oracle as RO

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
WAVE = {"rope_type": "wavelength", "factor": 8.0, "original_max_position_embeddings": 8192}
MROPE = {"rope_type": "default", "rope_theta": 10000000, "partial_rotary_factor": 0.25, "mrope_section": [11, 11, 10], "mrope_interleaved": True}


def plan(fp8lin, *args, **kw):
    return fp8lin.rotary_plan(*args, device="cpu", **kw)


def ints(p):
    return [s % 2 ** 64 for s in p.steps.tolist()]


def near(p, freq, axes=None):
    """The plan's steps within the roundings of the library's powers in 64 bits, a few half steps off each."""
    for j, (got, f) in enumerate(zip(ints(p), freq, strict=True)):
        assert got % 4 == (axes[j] if axes else 0)
        assert math.isclose((got - got % 4) / 2 ** 64, f / (2 * math.pi), rel_tol=64 * 2 ** -53, abs_tol=2 ** -62)


def test_theta_of_the_dict(fp8lin):
    for scaling in ({"rope_theta": 1e7}, {"rope_type": "default", "rope_theta": 1e7}, {"rope_theta": 1e7, "rope_type": "linear", "factor": 4.0},
                    {**YARN, "rope_theta": 1e7}, {**WAVE, "rope_theta": 1e7}):
        p = plan(fp8lin, 64, scaling=scaling)
        near(p, RO.frequencies(64, 1e7, scaling)[0])
        assert ints(plan(fp8lin, 64, 1e7, scaling)) == ints(p) == ints(plan(fp8lin, 64, theta=10000000, scaling={**scaling, "rope_theta": None}))
        for theta in (1e4, 1e7 + 1):
            with pytest.raises(fp8lin.Fp8linError):
                plan(fp8lin, 64, theta, scaling)
    # without either: 10000
    assert ints(plan(fp8lin, 64)) == ints(plan(fp8lin, 64, 1e4)) == ints(plan(fp8lin, 64, scaling={}))
    for bad in (0.0, -1.0, math.inf, math.nan, "base", [1e4]):
        with pytest.raises(fp8lin.Fp8linError):
            plan(fp8lin, 64, scaling={"rope_theta": bad})


def test_sections_of_the_dict(fp8lin):
    axes = [j % 3 if j % 3 and j < 3 * MROPE["mrope_section"][j % 3] else 0 for j in range(32)]
    assert set(axes) == {0, 1, 2}
    p = plan(fp8lin, 64, scaling=MROPE)
    near(p, RO.frequencies(64, 1e7)[0], axes)
    assert ints(p) == ints(plan(fp8lin, 64, 1e7, sections=[11, 11, 10])) == ints(plan(fp8lin, 64, 1e7, MROPE, sections=(11, 11, 10)))
    # a dict that does not say how its sections lie: the argument says it
    unsaid = {k: v for k, v in MROPE.items() if k != "mrope_interleaved"}
    assert ints(plan(fp8lin, 64, scaling=unsaid, sections=[11, 11, 10])) == ints(p)
    with pytest.raises(fp8lin.Fp8linError):
        plan(fp8lin, 64, scaling=unsaid)
    for kw in (dict(scaling=MROPE, sections=[10, 11, 11]), dict(scaling={**MROPE, "mrope_interleaved": False}),
               dict(scaling={**MROPE, "mrope_section": [16, 16]}), dict(scaling={**MROPE, "mrope_section": 11}),
               dict(scaling={"mrope_interleaved": False}, sections=[11, 11, 10])):
        with pytest.raises(fp8lin.Fp8linError):
            plan(fp8lin, 64, **kw)


def test_part_of_the_head(fp8lin):
    assert ints(plan(fp8lin, 64, scaling=MROPE, head_dim=256)) == ints(plan(fp8lin, 64, scaling=MROPE))
    assert ints(plan(fp8lin, 20, scaling={"partial_rotary_factor": 0.25}, head_dim=80)) == ints(plan(fp8lin, 20))
    assert ints(plan(fp8lin, 64, head_dim=128)) == ints(plan(fp8lin, 64))
    for rotary, kw in ((256, dict(scaling=MROPE, head_dim=256)), (64, dict(scaling=MROPE, head_dim=128)),
                       (64, dict(scaling={"partial_rotary_factor": 1.0}, head_dim=128)), (64, dict(head_dim=32)), (64, dict(head_dim=0)),
                       (64, dict(scaling={"partial_rotary_factor": 0.0})), (64, dict(scaling={"partial_rotary_factor": 1.5})),
                       (64, dict(scaling={"partial_rotary_factor": math.nan}))):
        with pytest.raises(fp8lin.Fp8linError):
            plan(fp8lin, rotary, **kw)


@pytest.mark.parametrize("of,all_dim", [(1.0, 1.0), (0.707, 0.707), (1.0, 0.5), (0.707, 1.0)])
def test_yarn_magnitude_of_two_scales(fp8lin, of, all_dim):
    """mscale and mscale_all_dim: the ratio of 0.1 m ln(factor) + 1 of the two; of a factor up to 1, 1."""
    scaling = {**YARN, "mscale": of, "mscale_all_dim": all_dim}
    want = (0.1 * of * math.log(40.0) + 1) / (0.1 * all_dim * math.log(40.0) + 1)
    p = plan(fp8lin, 64, 1e4, scaling)
    assert math.isclose(p.magnitude, want, rel_tol=1e-14) and ints(p) == ints(plan(fp8lin, 64, 1e4, YARN))
    assert plan(fp8lin, 64, 1e4, {**scaling, "factor": 0.5}).magnitude == 1.0
    assert plan(fp8lin, 64, 1e4, scaling, magnitude=1.5).magnitude == 1.5
    assert math.isclose(plan(fp8lin, 64, 1e4, YARN).magnitude, 0.1 * math.log(40.0) + 1, rel_tol=1e-14)


@pytest.mark.parametrize("scaling", [
    # one of the two scales: its meaning is not settled; both beside a magnitude of its own; none that are positive numbers
    {**YARN, "mscale": 0.707}, {**YARN, "mscale_all_dim": 1.0}, {**YARN, "mscale": 1.0, "mscale_all_dim": 0.0}, {**YARN, "mscale": -1.0, "mscale_all_dim": 1.0},
    {**YARN, "mscale": 1.0, "mscale_all_dim": 1.0, "attention_factor": 1.2}, {**WAVE, "mscale": 1.0, "mscale_all_dim": 1.0},
    # borders that are not rounded to whole pairs, or are nothing
    {**YARN, "truncate": False}, {**YARN, "beta_slow": 0}, {**YARN, "beta_fast": 0.0}, {**WAVE, "low_freq_factor": 0}, {**WAVE, "high_freq_factor": 0.0},
    # without a factor
    {"rope_type": "linear"}, {"rope_type": "ntk"}, {"rope_type": "linear", "factor": None}, {"rope_type": "yarn", "original_max_position_embeddings": 4096},
    {"rope_type": "wavelength", "original_max_position_embeddings": 4096},
    # keys of no form, or of another one
    {**YARN, "finetuned": True}, {"rope_type": "linear", "factor": 2.0, "long_factor": [1.0]}, {"rope_type": "default", "factor": 2.0}, {"factor": 2.0},
    {"rope_type": "linear", "factor": 2.0, "beta_fast": 32}, {**YARN, "low_freq_factor": 1.0}, {**WAVE, "beta_slow": 1.0}, {**WAVE, "truncate": True},
    {"full_attention": {"rope_type": "default"}}, {"scale": 2.0},
    # two types, no type, and values that are no numbers
    {**YARN, "type": "linear"}, {"rope_type": 4, "factor": 2.0}, {"rope_type": ["linear"], "factor": 2.0}, {**YARN, "factor": "many"},
    {**YARN, "beta_fast": [32]}, {**YARN, "attention_factor": "auto"}, {**YARN, "original_max_position_embeddings": "long"},
], ids=str)
def test_refused(fp8lin, scaling):
    with pytest.raises(fp8lin.Fp8linError):
        plan(fp8lin, 64, 1e4, scaling)


@pytest.mark.parametrize("scaling", ["yarn", [("rope_type", "yarn")], 4.0], ids=str)
def test_no_dict(fp8lin, scaling):
    with pytest.raises(fp8lin.Fp8linError):
        plan(fp8lin, 64, 1e4, scaling)


@pytest.mark.parametrize("scaling,as_", [
    ({"type": "linear", "factor": 4}, {"rope_type": "linear", "factor": 4.0}), ({**YARN, "type": "yarn"}, YARN), ({**YARN, "truncate": True}, YARN),
    ({**YARN, "truncate": None, "beta_fast": None, "mscale": None, "mscale_all_dim": None, "attention_factor": None}, YARN),
    ({**YARN, "beta_slow": 1, "beta_fast": 32}, YARN), ({**WAVE, "low_freq_factor": 1.0, "high_freq_factor": 4.0}, WAVE),
    ({"rope_type": "ntk", "factor": 2.0, "original_max_position_embeddings": 4096}, {"rope_type": "ntk", "factor": 2.0}),
    ({"rope_type": None, "type": None}, None), ({"rope_type": "default", "factor": None}, None),
], ids=str)
def test_read(fp8lin, scaling, as_):
    """Null values are those that are not there."""
    got, want = plan(fp8lin, 64, 1e4, scaling), plan(fp8lin, 64, 1e4, as_)
    assert ints(got) == ints(want) and got.magnitude == want.magnitude
