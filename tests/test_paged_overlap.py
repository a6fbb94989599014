"""Operands of the paged-cache operators that share memory, without a GPU: what the C ABI refuses before it touches a device."""
import pytest

# 16-byte aligned, never dereferenced: an accepted call ends at the device check.
A = 0x100000000


def accepted(rc):
    """Past validation: without a GPU the device check fails (3: unsupported, 5: device), with one nothing is called."""
    return rc not in (1, 2, 4)


LAYOUT = "lengths counts table table_ld free_pages free_count cursor requests width page_size tokens offsets new_lengths slots " \
         "positions new_table new_table_ld new_cursor workspace workspace_bytes stream".split()


def layout(fp8lin, **kw):
    d = dict(zip(LAYOUT, [A, A + 0x100, A + 0x1000, 8, A + 0x200, 10, A + 0x300, 3, 8, 16, 4, A + 0x400, A + 0x500, A + 0x600, A + 0x700,
                          A + 0x2000, 8, A + 0x800, A + 0x3000, 1 << 20, None]))
    d.update(kw)
    return fp8lin.lib().fp8lin_paged_layout(*[d[k] for k in LAYOUT])


@pytest.mark.parametrize("change", [
    dict(new_lengths=A), dict(new_lengths=A + 8), dict(new_lengths=A - 8), dict(new_lengths=A + 0x100), dict(new_cursor=A + 0x300),
    dict(new_cursor=A + 4), dict(new_cursor=A + 0x100), dict(offsets=A - 12), dict(offsets=A + 0x200 + 36), dict(slots=A + 0x1000 + 92),
    dict(positions=A + 0x600), dict(positions=A + 0x600 - 24), dict(new_table=A + 0x1000 + 32), dict(new_table=A + 0x1000 - 92),
    dict(new_table=A + 0x1000 + 4, new_table_ld=100), dict(new_table=A + 0x200), dict(new_table=A), dict(new_lengths=A + 0x2000 + 4),
    dict(new_table=A + 0x1000, new_lengths=A + 0x1000), dict(table_ld=20, new_cursor=A + 0x1000 + 80),
    dict(requests=1500, workspace=A + 0x100000, new_lengths=A + 0x100000),
], ids=str)
def test_layout_refuses_shared_memory(fp8lin, change):
    assert layout(fp8lin, **change) == 2
    assert b"overlaps" in fp8lin.lib().fp8lin_last_error()


@pytest.mark.parametrize("change", [
    {}, dict(new_table=A + 0x1000), dict(new_lengths=A + 12), dict(new_lengths=A - 12), dict(offsets=A - 16),
    dict(new_table=A + 0x1000 + 96), dict(new_table=A + 0x1000 - 96), dict(cursor=None), dict(tokens=0, slots=None, positions=None),
    # rows side by side in one buffer, a cursor between rows
    dict(table_ld=20, new_table=A + 0x1000 + 32, new_table_ld=20), dict(table_ld=20, new_table=A + 0x1000 - 32, new_table_ld=20),
    dict(table_ld=20, new_cursor=A + 0x1000 + 76), dict(table_ld=20, new_cursor=A + 0x1000 + 32),
], ids=str)
def test_layout_takes_what_is_apart(fp8lin, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the call would launch")
    assert accepted(layout(fp8lin, **change))


@pytest.mark.parametrize("change", [dict(table_ld=1 << 62), dict(new_table_ld=1 << 62), dict(table_ld=1 << 56)], ids=str)
def test_layout_refuses_strides_past_64_bits(fp8lin, change):
    assert layout(fp8lin, **change) == 1


VERIFY = "logits logits_f32 logits_ld draft_probs draft_ld prob_rows tokens uniforms offsets temperature requests rows vocab accepted " \
         "out workspace workspace_bytes stream".split()


def verify(fp8lin, **kw):
    d = dict(zip(VERIFY, [A, 0, 100, A + 0x10000, 100, 5, A + 0x20000, A + 0x21000, A + 0x22000, A + 0x23000, 2, 7, 100, A + 0x24000,
                          A + 0x25000, A + 0x30000, 1 << 30, None]))
    d.update(kw)
    return fp8lin.lib().fp8lin_verify_drafts(*[d[k] for k in VERIFY])


@pytest.mark.parametrize("change", [
    dict(out=A + 0x20000), dict(out=A + 0x20000 + 8), dict(out=A + 0x20000 - 8), dict(out=A + 0x21000), dict(out=A + 0x22000 - 48),
    dict(out=A), dict(out=A + 0x10000 + 1992), dict(accepted=A + 0x20000 + 52), dict(accepted=A + 0x22000 + 8), dict(accepted=A + 0x23000),
    dict(accepted=A + 0x25000), dict(out=A + 0x30000), dict(workspace=A + 0x20000), dict(workspace=A),
], ids=str)
def test_verify_refuses_shared_memory(fp8lin, change):
    assert verify(fp8lin, **change) == 2
    assert b"overlaps" in fp8lin.lib().fp8lin_last_error()


@pytest.mark.parametrize("change", [{}, dict(out=A + 0x20000 + 56), dict(accepted=A + 0x22000 + 12), dict(temperature=None),
                                    dict(draft_probs=None, out=A + 0x10000), dict(logits_ld=200, out=A + 216)], ids=str)
def test_verify_takes_what_is_apart(fp8lin, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the call would launch")
    assert accepted(verify(fp8lin, **change))


@pytest.mark.parametrize("change", [dict(logits_ld=1 << 62), dict(draft_ld=1 << 61), dict(prob_rows=1 << 40)], ids=str)
def test_verify_refuses_strides_past_64_bits(fp8lin, change):
    assert verify(fp8lin, **change) == 1
