"""A rule of synchronisation that no run can be relied on to show broken, read from the source of the attention behind a shared prefix."""
import re

from test_kv8_sync_host import _kernel


def test_a_share_s_q_is_seen_however_late_its_issuer_looks():
    """Where both halves of a CTA hold the same rows, all softmax warps announce each share's q, and both MMA issuers wait for it. An issuer
    without tiles in a share may be late: the softmax warps need nothing of it, and only that it leaves share i keeps back share i + 2. So when it
    looks for the q of share i, those of shares 0 .. i - 1 (it must wait) to 0 .. i + 1 (it must not) may have come in. A wait for
    parity p ends while the number of complete phases of its barrier is odd and p is 0, or even and p is 1."""
    k = _kernel("attn_kv8_shared_tc_kernel", "kv8_shared.cu")
    both = lambda e: re.sub(r"ALT \? ([^:()]+) : [^:()]+", r"\1", e)
    bar, parity = (both(e) for e in re.search(r"wait\(&q_full\[([^\]]+)\], (.+?)\);", k).groups())
    announced, = (both(e) for e in re.findall(r"mbar_arrive_if\(&q_full\[([^\]]+)\]", k))
    at = lambda e, i: int(eval(e, {"i": i, "sq": i}))  # of share i, which is also the number of q's before its
    for i in range(12):
        for came in (i, i + 1, i + 2):
            phases = sum(at(announced, x) == at(bar, i) for x in range(came))
            assert (phases % 2 != at(parity, i) % 2) == (came > i), (i, came)
