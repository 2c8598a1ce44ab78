"""Arguments that the experts' products and the draw of a class refuse. They are looked at before anything is launched, so no GPU is needed."""
import numpy as np
import pytest

import catboost_amd as cb

BUFFER = np.zeros(1 << 16, np.uint8)
AT = (BUFFER.ctypes.data + 255) & ~255  # never read or written: every call here is refused, or has nothing to do


@pytest.mark.parametrize("arguments,message", [
    (dict(value_type=4), "value type"), (dict(classes=0), "no classes"), (dict(classes=(1 << 24) + 1, stride=1 << 25), "too many classes"),
    (dict(scores=0), "scores pointer is null"), (dict(scores=AT + 2), "multiple of the value size"), (dict(stride=9), "shorter than a row"),
    (dict(rows=(1 << 40) + 1), "too many rows"), (dict(rows=1 << 40, stride=1 << 30), "too large"), (dict(uniform=0), "uniform pointer is null"),
    (dict(indexes=0), "indexes pointer is null"), (dict(), "memory that a GPU can write"),
])
def test_sample_classes(arguments, message):
    a = dict(dict(value_type=cb.FLOAT32, rows=4, classes=10, scores=AT, stride=10, uniform=AT, indexes=AT), **arguments)
    with pytest.raises(cb.CatBoostError, match=message):
        cb.sample_classes(a["value_type"], a["rows"], a["classes"], a["scores"], a["stride"], cb.sampling(), a["uniform"], a["indexes"], AT, AT, 1 << 15)


def test_sample_classes_without_a_struct():
    assert not cb.load_library().CbHipSampleClasses(cb.FLOAT32, 1, 1, AT, 1, None, AT, AT, AT, AT, 0, None)
    assert "sampling is null" in cb.last_error()


def test_sample_classes_with_nothing_to_do():
    cb.sample_classes(cb.FLOAT32, 0, 10, 0, 10, cb.sampling(), 0, 0)
    assert cb.sample_classes_bytes(9, 4, 10) == 0 and cb.sample_classes_bytes(cb.FLOAT32, 0, 10) == 0


ROUTED = [
    (dict(value_type=5), "value type"), (dict(experts=0), "experts: 0"), (dict(experts=1025), "experts: 1025"), (dict(offsets=0), "offsets pointer is null"),
    (dict(rows=1 << 31), "too many rows"), (dict(width=1 << 30), "too wide"), (dict(outputs=1 << 30), "too many outputs"), (dict(weights=0), "pointer is null"),
    (dict(expert_stride=31), "shorter than an expert"), (dict(stride=3), "shorter than a row"), (dict(source=0), "pointer is null"),
    (dict(result=0), "pointer is null"), (dict(weights=AT + 1), "multiple of the value size"), (dict(), "GPU can write"),
]


@pytest.mark.parametrize("arguments,message", ROUTED)
@pytest.mark.parametrize("call", ["multiply", "multiply_backward", "gated", "gated_backward"])
def test_products(arguments, message, call):
    a = dict(dict(value_type=cb.BFLOAT16, rows=4, width=8, outputs=4, experts=3, offsets=AT, source=AT, stride=8, weights=AT, expert_stride=32,
                  result=AT + 4096), **arguments)
    head = a["rows"], a["width"], a["outputs"], a["experts"], a["offsets"]
    kind, x, w, es, y, st = a["value_type"], a["source"], a["weights"], a["expert_stride"], a["result"], a["stride"]
    with pytest.raises(cb.CatBoostError, match=message):
        if call == "multiply":
            cb.multiply_rows(kind, *head, x, st, w, es, y, st)
        elif call == "multiply_backward":
            cb.multiply_rows_backward(kind, *head, y, st, x, st, w, es, AT + 8192, st, w and w + 512, es)
        elif call == "gated":
            cb.gated_rows(kind, cb.SILU, *head, x, st, w, w, es, y, st)
        else:
            cb.gated_rows_backward(kind, cb.SILU, *head, y, st, x, st, w, w, es, AT + 1024, AT + 2048, AT + 8192, st, w and w + 512, w and w + 1024, es)


@pytest.mark.parametrize("activation", [-1, 4])
def test_unknown_activations(activation):
    with pytest.raises(cb.CatBoostError, match="unknown activation"):
        cb.gated_rows(cb.FLOAT32, activation, 4, 8, 4, 1, 0, AT, 8, AT, AT, 32, AT, 4)
    with pytest.raises(cb.CatBoostError, match="unknown activation"):
        cb.gated_rows_backward(cb.FLOAT32, activation, 4, 8, 4, 1, 0, AT, 4, AT, 8, AT, AT, 32, AT, AT, AT, 8, AT, AT, 32)


def test_what_the_gradients_of_a_gate_need():
    def call(kept=AT, pre=AT, dgate=AT, dup=AT):
        cb.gated_rows_backward(cb.FLOAT32, cb.SILU, 4, 8, 4, 1, 0, AT, 4, AT, 8, AT, AT, 32, kept, pre, AT, 8, dgate, dup, 32)

    for arguments, message in ((dict(kept=0), "kept values pointer is null"), (dict(pre=0), "gate and up gradients pointer is null"),
                               (dict(dgate=0), "one projection alone"), (dict(dup=0), "one projection alone"), (dict(kept=AT + 2), "multiple of the value size")):
        with pytest.raises(cb.CatBoostError, match=message):
            call(**arguments)
    with pytest.raises(cb.CatBoostError, match="kept values pointer"):
        cb.gated_rows(cb.FLOAT32, cb.SILU, 4, 8, 4, 1, 0, AT, 8, AT, AT, 32, AT, 4, AT + 2)


def test_gradients_of_16_bits_in_place_of_kept_values():
    with pytest.raises(cb.CatBoostError, match="memory of their own"):
        cb.gated_rows_backward(cb.FLOAT16, cb.SILU, 4, 8, 4, 1, 0, AT, 4, AT, 8, AT, AT, 32, AT + 512, AT + 512, AT, 8, AT, AT, 32)


def test_products_with_nothing_to_do():
    cb.multiply_rows(cb.FLOAT32, 0, 8, 4, 2, AT, 0, 8, 0, 32, 0, 4)
    cb.multiply_rows(cb.FLOAT32, 4, 8, 0, 2, AT, 0, 8, 0, 32, 0, 4)
    cb.gated_rows(cb.FLOAT32, cb.RELU, 0, 8, 4, 2, AT, 0, 8, 0, 0, 32, 0, 4)
    cb.multiply_rows_backward(cb.FLOAT32, 4, 8, 4, 2, AT, 0, 4, 0, 8, 0, 32, 0, 8, 0, 32)  # neither gradient is wanted
    cb.multiply_rows_backward(cb.FLOAT32, 0, 8, 4, 2, AT, 0, 4, 0, 8, 0, 32, AT, 8, 0, 32)
    cb.gated_rows_backward(cb.FLOAT32, cb.RELU, 0, 8, 4, 2, AT, 0, 4, 0, 8, 0, 0, 32, 0, 0, AT, 8, 0, 0, 32)
