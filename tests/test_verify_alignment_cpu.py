"""Pointers that are not aligned to their types are refused before anything reaches a device."""
import pytest

P = 1 << 20                                            # a pointer that nothing follows


@pytest.mark.parametrize("name", ["first", "tokens", "temperature", "accepted", "next"])
@pytest.mark.parametrize("by", [1, 2, 3])
def test_verify(pkg, name, by):
    fields = dict(sequences=2, rows=5, first=P, tokens=P, logits=P, ld=50, temperature=P, random=P)
    outs = {"accepted": P, "next": P}
    (fields if name in fields else outs)[name] += by
    assert pkg.lib.cmlb200_verify_drafts(pkg.Drafts(**fields), P, 0, 50, 50, outs["accepted"], outs["next"], P, None) == -1
    assert b"aligned" in pkg.last_error()
