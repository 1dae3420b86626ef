"""CPU: what verifying drafts within a limit of positions refuses before any
device use (as test_drafts_api)."""
import pytest

from test_drafts_api import RIGHT, refused, verify


def test_limits():
    for limit in (0, 1, 1 << 31, (1 << 32) - 1, 1 << 32, 1 << 40):
        refused(RIGHT, verify, pos_limit=limit)
    refused("negative", verify, pos_limit=-1)
    for limit in (0, (1 << 32) - 1):
        refused("a limit of positions without positions", verify, pos_limit=limit, pos=None)
    refused(RIGHT, verify, pos_limit=1 << 32, pos=None)
    refused(RIGHT, verify, pos_limit=None, pos=None)
