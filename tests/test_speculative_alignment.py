"""Unaligned words are refused by the speculative entry points before anything
runs (no GPU: a call that passed the checks would report a failed step)."""
import ctypes

import pytest

import charlotte_b200 as cb


def status(entry, args):
    return getattr(cb.lib(), f"cb_{entry}_run")(ctypes.byref(args), 0, None), cb.last_error()


def cache():
    return cb.Cache(format=cb.CACHE_F16, slots=16, kv_heads=2, head_dim=64, key=4096, value=8192)


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("entry,field", [*(("verify", f) for f in ("ids", "uniforms", "path", "kept", "sampled", "nodes")),
                                         *(("cache_write", f) for f in ("turns", "factors", "lengths", "nodes")),
                                         *(("cache_keep", f) for f in ("path", "kept", "lengths", "new_lengths")),
                                         *(("cache_read", f) for f in ("starts", "lengths"))])
def test_words_are_aligned(entry, field, by):
    args = {"verify": lambda: cb.Verify(candidates=4096, ids=4096, uniforms=4096, path=4096, kept=4096, sampled=4096, sequences=1, tokens=1),
            "cache_write": lambda: cb.CacheWrite(cache=cache(), key=4096, value=4096, turns=4096, sequences=1, tokens=1),
            "cache_keep": lambda: cb.CacheKeep(cache=cache(), path=4096, kept=4096, sequences=1, tokens=1, layers=1),
            "cache_read": lambda: cb.CacheRead(cache=cache(), out_key=4096, sequences=1, tokens=1)}[entry]()
    setattr(args, field, 4096 + by)
    rc, message = status(entry, args)
    assert rc == cb.ERROR_INVALID and "unaligned" in message, message
