"""Arguments that the operators on scores and rows refuse. They are looked at before anything is launched, so no GPU is needed."""
import numpy as np
import pytest

import catboost_amd as cb

BUFFER = np.zeros(1 << 16, np.uint8)
AT = (BUFFER.ctypes.data + 255) & ~255  # never read or written: every call here is refused, or has nothing to do


def adjust(value_type=cb.FLOAT32, rows=4, classes=10, scores=AT, score_stride=10, result=AT + 8192, result_stride=10, **parts):
    cb.adjust_scores(value_type, rows, classes, scores, score_stride, cb.score_adjustment(**parts), result, result_stride)


@pytest.mark.parametrize("arguments,message", [
    (dict(value_type=4), "value type"), (dict(value_type=-1), "value type"),
    (dict(scores=0), "scores pointer is null"), (dict(result=0), "result pointer is null"),
    (dict(score_stride=9), "shorter than a row"), (dict(result_stride=9), "shorter than a row"),
    (dict(scores=AT + 2), "multiple of the value size"), (dict(classes=1 << 31, score_stride=1 << 31, result_stride=1 << 31), "too many classes"),
    (dict(rows=1 << 59), "too large"),
    (dict(result=AT, result_stride=12), "same stride"),
    (dict(history_offsets_ptr=AT, history_count=3), "history pointer is null"), (dict(history_ptr=AT, history_count=3), "history offsets"),
    (dict(bias_offsets_ptr=AT, bias_classes_ptr=AT, bias_count=1), "bias classes or values"), (dict(bias_values_ptr=AT), "bias offsets"),
    (dict(bias_offsets_ptr=AT, bias_classes_ptr=AT, bias_values_ptr=AT, bias_count=1 << 31), "too many biases"),
    (dict(class_bias_ptr=AT, class_bias_stride=9), "class bias stride"),
    (dict(allowed_ptr=AT, allowed_count=4, allowed_stride=0), "mask stride"), (dict(allowed_ptr=AT, allowed_count=3, allowed_stride=1), "fewer masks"),
    (dict(allowed_rows_ptr=AT), "mask pointer is null"),
    (dict(), "memory that a GPU can write"),  # all in order, but for host memory
])
def test_adjust_scores(arguments, message):
    with pytest.raises(cb.CatBoostError, match=message):
        adjust(**arguments)


def test_adjust_scores_with_nothing_to_do():
    adjust(rows=0)
    adjust(classes=0, score_stride=0, result_stride=0)


def test_adjust_scores_without_a_struct():
    assert not cb.load_library().CbHipAdjustScores(cb.FLOAT32, 1, 1, AT, 1, None, AT, 1, None)
    assert "adjustment is null" in cb.last_error()


@pytest.mark.parametrize("arguments,message", [
    (dict(value_type=7), "value type"), (dict(classes=1025, stride=1025), "at most 1024"), (dict(count=0), "1 to 32"), (dict(count=33), "1 to 32"),
    (dict(classes=0), "no classes"), (dict(scores=0), "scores pointer is null"), (dict(indexes=0), "pointer is null"),
    (dict(weights=0), "pointer is null"), (dict(stride=9), "shorter than a row"), (dict(rows=1 << 49), "too many rows"), (dict(), "GPU can write"),
])
@pytest.mark.parametrize("backward", [False, True])
def test_select_top(arguments, message, backward):
    a = dict(dict(value_type=cb.FLOAT32, rows=4, classes=10, scores=AT, stride=10, count=2, indexes=AT, weights=AT), **arguments)
    with pytest.raises(cb.CatBoostError, match=message):
        if backward:
            cb.select_top_backward(a["value_type"], a["rows"], a["classes"], a["scores"], a["stride"], a["count"], False, a["indexes"], a["weights"],
                                   AT, AT, max(a["classes"], 10))
        else:
            cb.select_top(a["value_type"], a["rows"], a["classes"], a["scores"], a["stride"], a["count"], False, a["indexes"], a["weights"])


def test_select_top_with_nothing_to_do():
    cb.select_top(cb.FLOAT32, 0, 10, 0, 0, 2, True, 0, 0)
    cb.select_top_backward(cb.FLOAT32, 0, 10, 0, 0, 2, True, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("arguments,message", [
    (dict(experts=0), "experts: 0"), (dict(experts=1025), "experts: 1025"), (dict(slots=1 << 31), "too many slots"), (dict(ids=0), "ids or places"),
    (dict(places=0), "ids or places"), (dict(offsets=0), "offsets pointer"), (dict(workspace=0), "workspace"), (dict(size=-1), "are needed"),
    (dict(workspace=AT + 1), "multiple of 4"), (dict(), "GPU can write"),
])
def test_sort_by_expert(arguments, message):
    a = dict(dict(slots=100, experts=8, ids=AT, places=AT, offsets=AT, workspace=AT, size=0), **arguments)
    needed = cb.sort_by_expert_bytes(a["slots"], a["experts"])
    with pytest.raises(cb.CatBoostError, match=message):
        cb.sort_by_expert(a["slots"], a["experts"], a["ids"], a["places"], a["offsets"], a["workspace"], needed + a["size"])


ROUTED = [
    (dict(value_type=5), "value type"), (dict(per_row=0), "slots per row: 0"), (dict(per_row=65), "slots per row: 65"), (dict(places=0), "places pointer"),
    (dict(width=1 << 31, stride=1 << 31), "too wide"), (dict(rows=(1 << 40) + 1), "too many rows"), (dict(sorted_rows=1 << 31), "too many sorted rows"),
    (dict(plain=0), "pointer is null"), (dict(sorted=0), "pointer is null"), (dict(stride=7), "shorter than a row"), (dict(), "GPU can write"),
]


@pytest.mark.parametrize("arguments,message", ROUTED)
@pytest.mark.parametrize("call", ["dispatch", "combine", "backward"])
def test_routed_rows(arguments, message, call):
    a = dict(dict(value_type=cb.BFLOAT16, rows=4, width=8, per_row=2, plain=AT, stride=8, places=AT, sorted=AT + 4096, sorted_rows=8), **arguments)
    with pytest.raises(cb.CatBoostError, match=message):
        if call == "dispatch":
            cb.dispatch_rows(a["value_type"], a["rows"], a["width"], a["per_row"], a["plain"], a["stride"], a["places"], a["sorted"], a["sorted_rows"], a["stride"])
        elif call == "combine":
            cb.combine_rows(a["value_type"], a["rows"], a["width"], a["per_row"], a["sorted"], a["sorted_rows"], a["stride"], a["places"], 0, a["plain"],
                            a["stride"])
        else:
            cb.combine_rows_backward(a["value_type"], a["rows"], a["width"], a["per_row"], a["plain"], a["stride"], a["sorted"], a["sorted_rows"],
                                     a["stride"], a["places"], 0, AT + 16384, a["stride"], AT + 32768)


def test_routed_rows_with_nothing_to_do():
    cb.dispatch_rows(cb.FLOAT32, 0, 8, 2, 0, 8, 0, 0, 8, 8)
    cb.dispatch_rows(cb.FLOAT32, 4, 8, 2, 0, 8, 0, 0, 0, 8)
    cb.combine_rows(cb.FLOAT32, 0, 8, 2, 0, 8, 8, 0, 0, 0, 8)
    cb.combine_rows(cb.FLOAT32, 4, 0, 2, 0, 8, 8, 0, 0, 0, 8)
    cb.combine_rows_backward(cb.FLOAT32, 0, 8, 2, 0, 8, 0, 8, 8, 0, 0, 0, 8, 0)
    cb.combine_rows_backward(cb.FLOAT32, 4, 8, 2, 0, 8, 0, 8, 8, 0, 0, 0, 8, 0)  # neither gradient is wanted


def test_workspace_sizes():
    assert cb.sort_by_expert_bytes(0, 8) > 0
    assert cb.sort_by_expert_bytes(100, 0) == 0 and cb.sort_by_expert_bytes(1 << 31, 8) == 0


def test_eval_routed_without_evaluators():
    with pytest.raises(cb.CatBoostError, match="evaluators: 0"):
        cb.eval_routed_bytes([], cb.LAYOUT_FLAT_ROWS, 10, 1)
    with pytest.raises(cb.CatBoostError, match="evaluators: 0"):
        cb.eval_routed([], cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, AT, 4), 10, 1, AT, 0, AT, AT, 1 << 20)


def test_eval_routed_with_a_closed_evaluator():
    class Closed:
        _h = None

    with pytest.raises(cb.CatBoostError, match="handle is null"):
        cb.eval_routed_bytes([Closed()], cb.LAYOUT_FLAT_ROWS, 10, 1)
    with pytest.raises(cb.CatBoostError, match="handle is null"):
        cb.eval_routed([Closed(), Closed()], cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, AT, 4), 10, 1, AT, 0, AT, AT, 1 << 20)
