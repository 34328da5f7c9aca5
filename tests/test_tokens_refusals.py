"""Refusals of the token and 4-bit entries that depend on another argument, and what their messages say (no device call
is made)."""
from __future__ import annotations

from stand_in import launched
from test_tokens_contract import P, S, refusal


def test_maps_alone_have_no_width(tmp_path):
    calls = [["sort_tokens", dict(expert_ids=P, offsets=P, route_pos=P, sorted_route=P, tokens=tokens, experts=3, top_k=2, **hidden)]
             for tokens in (4, 3000, 20000) for hidden in ({}, dict(hidden=0), dict(hidden=-1))]
    assert all(launched(tmp_path, calls)[0])
    for hidden in (0, -1):
        assert refusal("sort_tokens", hidden=hidden) == S.kInvalidArgument  # (with rows)
