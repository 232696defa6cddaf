"""Plan scratch of the decoding operators for a device other than the current one: its own SM count, by its ordinal."""
from types import SimpleNamespace

import torch

from augur_v100_b200 import host, kv


def test_scratch_for_another_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda ordinal: SimpleNamespace(multi_processor_count=(132, 148)[ordinal]))
    assert host.sm_count() == host.sm_count(0) == 132 and host.sm_count(1) == 148
    for scratch in (lambda sms: kv.paged_attention_scratch_bytes(24, 4, 256, 1, sms), lambda sms: host.logprobs_scratch_bytes(8, 20, sms)):
        assert scratch(0) == scratch(132) < scratch(host.sm_count(1)) == scratch(148)
