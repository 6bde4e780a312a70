"""Comparisons that hold a value only where it is shown to be near: a NaN, or an infinity, is never within a limit, and where the
reference is one the value has to be the same."""

import numpy as np
import torch

from tree_cases import attention, attention_limit, lse_limit


def within(got, ref, limit, what="value"):
    """Every value of got: at most limit from a finite reference, equal to one that is not (NaN to NaN)."""
    got, ref, limit = np.broadcast_arrays(np.asarray(got, np.float64), np.asarray(ref, np.float64), np.asarray(limit, np.float64))
    finite = np.isfinite(ref)
    assert np.isfinite(limit[finite]).all(), f"{what}: no limit"
    with np.errstate(invalid="ignore"):
        near = np.abs(got - ref) <= limit
    same = np.where(finite, near, (got == ref) | np.isnan(got) & np.isnan(ref))
    if not same.all():
        at = tuple(int(i) for i in np.argwhere(~same)[0])
        raise AssertionError(f"{what}: {int((~same).sum())} of {same.size} off, at {at} {got[at]} in place of {ref[at]} +- {limit[at]}")


def same_attention(case, out, lse, scale=None):
    """Every token of a row of a tree attention case (test_gpu_tree.Case) against the definition; values of V that are not finite
    reach the outputs that see them."""
    with np.errstate(invalid="ignore"):
        ref, ref_lse, size, most = attention(case.q, case.cache, case.qo, case.kvp, case.ids, case.last, case.masks, scale)
    keys = max([1, *(b - a for a, b in zip(case.kvp[:-1], case.kvp[1:]))]) * case.page
    T = case.qo[-1]  # tokens of no row are behind
    got, got_lse = out.detach().cpu().double().numpy()[:T], lse.cpu().double().numpy()[:T]
    ref, ref_lse, size, most = ref[:T], ref_lse[:T], size[:T], most[:T]
    assert not np.isnan(ref_lse).any()
    blind = np.isneginf(ref_lse)
    assert (got[blind] == 0).all()
    with np.errstate(invalid="ignore"):
        limit = np.where(blind[..., None], 0, attention_limit(ref, np.where(blind[..., None], 0, size), most, out.dtype, keys, ref.shape[2]))
        within(got, ref, limit, "out")
        within(got_lse, ref_lse, lse_limit(ref_lse, most, keys, ref.shape[2]), "lse")


def same_logits(out, ref, touched, size, before):
    """Adjusted logits against the definition (tree_cases.adjusted): half a step of the output's type, and 8 * 2^-24 of the largest
    magnitude on the way (a quotient or product, the frequency's product and sum, presence and bias round once each); rows of no
    request to the last bit. What is past the type's largest value is infinite, or that value where it lies that near."""
    raw = lambda t: t.detach().contiguous().cpu().numpy() if t.dtype == torch.float32 else t.detach().contiguous().cpu().view(torch.int16).numpy()
    assert np.array_equal(raw(out).view(np.uint8).reshape(*out.shape, -1)[~touched], raw(before).view(np.uint8).reshape(*out.shape, -1)[~touched])
    got = out.detach().cpu().double().numpy()
    big, half = float(torch.finfo(out.dtype).max), torch.finfo(out.dtype).eps / 2
    ref, size = ref[touched], np.asarray(size)[touched]
    with np.errstate(invalid="ignore"):
        limit = half * np.abs(ref) + 8 * 2.0 ** -24 * size * (1 + half) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    far = np.isfinite(ref) & (np.abs(ref) >= big * (1 - half))
    got = got[touched]
    got = np.where(far & np.isinf(got) & (np.sign(got) == np.sign(ref)), ref, got)
    within(got, ref, limit, "logits")
