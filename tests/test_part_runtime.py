"""The parts' Runtime by position: a field that is added later goes behind those that callers may name by place."""
import torch

from damendaemon_b200.parts.interfaces import Runtime
from damendaemon_b200.parts.paged_attention import AttentionTuning


def test_fields_keep_their_places():
    tuning = AttentionTuning()
    runtime = Runtime(torch.bfloat16, torch.device("cpu"), "simt", "rows", tuning, 32)
    assert (runtime.page_size, runtime.attention_tuning, runtime.feed_forward) == (32, tuning, "auto")
    assert Runtime(torch.bfloat16, torch.device("cpu"), "auto", "auto", tuning, 16, "mx4").feed_forward == "mx4"
