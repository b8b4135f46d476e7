"""Refusals of the token mixer's C ABI that need no GPU."""
import ctypes as C

import pytest

from mixer_abi import Heads, Problem, library


@pytest.mark.parametrize("tokens", [2 ** 30 + 1, 2 ** 31 - 1])
def test_more_tokens_than_32_bits_can_place_are_refused(tokens):
    lib, one = library(), Heads(None, 1, 1, 1, 1)
    problem = Problem(1, tokens, 1, 1, 1, 0, one, one, one, None, None, 1.0)
    for call in (lambda: lib.rxmet_decayed_attention_forward(C.byref(problem), None, None, None, None, C.c_size_t(0), None),
                 lambda: lib.rxmet_decayed_attention_backward(C.byref(problem), None, None, None, None, None, None, None, None, C.c_size_t(0), None)):
        assert call() != 0 and b"tokens, at most" in lib.rxmet_last_error()


def test_a_wait_that_ran_out_is_reported(monkeypatch):
    import rx_met_b200
    from rx_met_b200 import _cabi

    class Fake:
        word, status = 0, 0

        def rxmet_wait_status(self, at):
            at._obj.value = self.word
            return self.status

        def rxmet_last_error(self):
            return b"no device"

    fake = Fake()
    monkeypatch.setattr(_cabi, "load_library", lambda: fake)
    assert rx_met_b200.wait_gave_up() is False
    fake.word = 1
    assert rx_met_b200.wait_gave_up() is True
    fake.status = -2
    with pytest.raises(RuntimeError, match="no device"):
        rx_met_b200.wait_gave_up()
