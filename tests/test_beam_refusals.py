"""CPU tests of what kvc_beam_select refuses.  The context is host-only: a call whose
arguments are all right ends with KVC_ERR_NO_DEVICE, so nothing runs."""
import pytest

import kvc

X, S, OS, OB, OT = 0x100000, 0x10000, 0x20000, 0x30000, 0x40000
GOOD = dict(logits=X, n_groups=2, n_beams=4, vocab=1000, n_out=8, out_scores=OS, out_beams=OB, out_tokens=OT, scores=S)


@pytest.fixture(scope="module")
def ctx():
    with kvc.Context(device=-1, pool_blocks=1, n_ssm_layers=0, max_seqs=1, max_seq_len=32, snapshot_slots=0) as c:
        yield c


def code(ctx, **over):
    with pytest.raises(kvc.KvcError) as e:
        ctx.beam_select(**{**GOOD, **over})
    return e.value.code


@pytest.mark.parametrize("over", [
    {}, {"scores": None}, {"row_stride": 1001}, {"dtype": kvc.DTYPE_BF16, "logits": X + 2}, {"logits": X + 4},
    {"n_out": 4, "out_scores": S}, {"n_beams": 64, "n_out": 128}, {"vocab": 1, "n_out": 128}, {"n_groups": 1, "vocab": 200000, "n_beams": 64},
    {"out_scores": X - 64}, {"out_tokens": X + 8 * 4000}, {"scores": X - 32},
])
def test_allowed(ctx, over):
    assert code(ctx, **over) == kvc.KVC_ERR_NO_DEVICE


@pytest.mark.parametrize("over", [
    {"logits": None}, {"out_scores": None}, {"out_beams": None}, {"out_tokens": None},
    {"dtype": 2}, {"dtype": -1}, {"n_groups": 0}, {"n_beams": 0}, {"vocab": 0}, {"n_out": 0}, {"n_out": -1}, {"n_groups": -3},
    {"row_stride": 999}, {"row_stride": -1}, {"logits": X + 2}, {"dtype": kvc.DTYPE_BF16, "logits": X + 1},
    {"scores": S + 2}, {"out_scores": OS + 1}, {"out_beams": OB + 2}, {"out_tokens": OT + 3},
    {"out_scores": X}, {"out_beams": X - 60}, {"out_tokens": X + 8 * 4000 - 4}, {"out_scores": OB + 60}, {"out_tokens": OB},
    {"out_tokens": OS}, {"out_scores": S}, {"out_beams": S}, {"n_out": 4, "out_tokens": S},
])
def test_refused(ctx, over):
    assert code(ctx, **over) == kvc.KVC_ERR_INVALID


@pytest.mark.parametrize("over", [
    {"n_beams": 65}, {"n_out": 129}, {"n_groups": 2**31 - 1, "n_beams": 2}, {"row_stride": 2**62},
    {"n_groups": 1, "n_beams": 64, "vocab": 2**31 - 1},
])
def test_out_of_range(ctx, over):
    assert code(ctx, **over) == kvc.KVC_ERR_RANGE


def test_null_context():
    assert kvc.lib().kvc_beam_select(None, X, 0, 1000, 2, 4, 1000, S, 8, OS, OB, OT, None) == kvc.KVC_ERR_INVALID
