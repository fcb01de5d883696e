"""CPU-only checks of the operators around drafted tokens and shared blocks: refusals beside those of test_drafts_host.py."""
from tests.test_drafts_host import INVALID, rotate


def test_rotate_refuses_heads_over_each_other_in_any_layout():
    at = 1 << 20
    # bf16, heads of 64 (128 bytes): queries, keys and values of four heads in turn, three tokens
    token = dict(q=at, qt=4 * 192, qh=192, hq=4, k=at + 128, kt=4 * 192, kh=192, hk=4, T=3)
    head = dict(q=at, qt=64, qh=3 * 192, hq=4, k=at + 384, kt=64, kh=3 * 192, hk=4, T=3)
    for lay, slot in ((token, 128), (head, 384)):
        strides = dict(qot=lay["qt"], qoh=lay["qh"], kot=lay["kt"], koh=lay["kh"])
        for bad in (dict(qo=at + slot, ko=at + 2 * slot), dict(qo=at, ko=at), dict(qo=at + 2 * slot, ko=at + 2 * slot), dict(qo=at + 2, ko=at + slot),
                    dict(qo=at, ko=at + slot + 64), dict(qo=at + 2 * slot, ko=at + 3 * slot - 2), dict(qo=at + 2 * slot - 2, ko=at + slot)):
            assert rotate(**lay, **strides, **bad) == INVALID, (lay, bad)
