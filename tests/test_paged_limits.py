"""Sizes past what a launch can count are refused before any device work."""
import pytest

from test_paged_args import S, plan, refused


@pytest.mark.parametrize("max_tok", [(1 << 31) + 1, 0xFFFFFF01, 0xFFFFFFFF])
def test_plan_rows(flh, max_tok):
    refused(flh, flh.ERR_UNSUPPORTED, "max_tok", flh.kv_plan, plan(flh, max_tok=max_tok), S)
