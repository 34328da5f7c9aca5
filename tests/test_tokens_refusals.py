"""Refusals of the token and 4-bit entries that depend on another argument, and what their messages say (no device call
is made)."""
from __future__ import annotations

import pytest

import raggedroute_amd as rr
from stand_in import launched
from test_tokens_contract import ENTRIES, P, S, ctx, refusal


def test_maps_alone_have_no_width(tmp_path):
    calls = [["sort_tokens", dict(expert_ids=P, offsets=P, route_pos=P, sorted_route=P, tokens=tokens, experts=3, top_k=2, **hidden)]
             for tokens in (4, 3000, 20000) for hidden in ({}, dict(hidden=0), dict(hidden=-1))]
    assert all(launched(tmp_path, calls)[0])
    for hidden in (0, -1):
        assert refusal("sort_tokens", hidden=hidden) == S.kInvalidArgument  # (with rows)


@pytest.mark.parametrize("name", list(ENTRIES))
def test_messages_speak_of_no_other_operator(name):
    """Whatever these entries share with the expert block's."""
    args, good = ENTRIES[name]
    contexts = [(ctx(architecture=int(rr.DeviceArchitecture.kSm86)), {}), (ctx(), dict(kernel=rr.kernel(rr.KernelFamily.kAuto, 1)))]
    if name == "sort_tokens":
        contexts.append((ctx(workspace=P + 4, workspace_bytes=1 << 20), dict(tokens=8193)))
    for context, change in contexts:
        status = getattr(rr, name)(args(**(good | change)), context)
        assert not status.ok() and "expert block" not in str(status.message)
