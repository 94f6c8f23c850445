"""kernels.act_format: the format that a block leaves behind."""
import threading

import pytest

from onedc_amd import kernels as K


def test_one_object_entered_inside_its_own_block():
    assert K.act() == K.DEFAULT_ACT
    other = "bf16" if K.DEFAULT_ACT == "f16" else "f16"
    a, b = K.act_format(other), K.act_format(K.DEFAULT_ACT)
    with a:
        with a:
            assert K.act() == other
            with b:
                assert K.act() == K.DEFAULT_ACT
                with a:
                    assert K.act() == other
                assert K.act() == K.DEFAULT_ACT
            assert K.act() == other
        assert K.act() == other
    assert K.act() == K.DEFAULT_ACT
    with pytest.raises(KeyError):
        with a:
            with a:
                raise KeyError("out of both blocks")
    assert K.act() == K.DEFAULT_ACT


def test_one_object_in_two_threads():
    other = "bf16" if K.DEFAULT_ACT == "f16" else "f16"
    a, seen, inside, leave = K.act_format(other), [], threading.Event(), threading.Event()

    def run():
        with K.act_format(other):
            with a:
                inside.set()
                leave.wait(30)
            seen.append(K.act())

    t = threading.Thread(target=run)
    with a:                                              # (the other thread's entry comes between this block's ends)
        t.start()
        assert inside.wait(30)
    assert K.act() == K.DEFAULT_ACT
    leave.set()
    t.join()
    assert seen == [other]


def test_a_format_that_does_not_exist_changes_nothing():
    with pytest.raises(ValueError):
        with K.act_format("fp8"):
            pass
    with K.act_format("bf16"):
        pass
    assert K.act() == K.DEFAULT_ACT


def test_as_a_decorator():
    @K.act_format("bf16")
    def depth(n):
        return [K.act()] + (depth(n - 1) if n else [])
    assert depth(3) == ["bf16"] * 4 and K.act() == K.DEFAULT_ACT
