"""Which devices the library takes: a yes is kept for the process, a no (which a
device query that failed gives too) is asked for again."""
import types

import torch

from burn_dragon_amd import recurrent


def test_a_failed_query_is_asked_again(monkeypatch):
    answers = [0, 0, 1]
    asked = []

    def supports_backend():
        asked.append(1)
        return answers.pop(0)

    monkeypatch.setattr(recurrent._lib, "load", lambda: types.SimpleNamespace(bdh_supports_backend=supports_backend))
    monkeypatch.setattr(recurrent, "_call_on", lambda device, fn, *args: fn(*args))
    # (of an index that no other test's tensors have)
    one, other = torch.device("cuda", 61), torch.device("cuda", 62)
    try:
        assert [recurrent._supported(one) for _ in range(5)] == [False, False, True, True, True]
        assert len(asked) == 3
        answers.append(0)
        assert not recurrent._supported(other)   # a device's own answer
        assert not recurrent._supported(torch.device("cpu")) and len(asked) == 4
    finally:
        for cached in (one, other):
            getattr(recurrent, "_supported_devices", set()).discard(cached)
