"""A launch holds fewer than 2^32 threads (a larger grid is cut off without an error): calls that need more are refused,
whatever the workgroups' size (no GPU needed)."""
from test_kv_refusals import FAKE, attend_call

ARGS = dict(H=16, Hkv=16, hd=128, q_stride=0, page=64, scratch=FAKE, scratch_bytes=1 << 62)


def test_workgroups_of_512_threads():
    """256 new tokens of 16 heads in each of 2^18 sequences: 2^23 workgroups of eight waves."""
    st, err = attend_call(T=1 << 26, B=1 << 18, cu=FAKE, max_len=1 << 14, max_new=256, **ARGS)
    assert st == -1 and "uwc_kv_attend: too many tokens" in err


def test_workgroups_of_256_threads():
    """A token of 16 heads in each of 2^20 sequences: 2^24 workgroups of four waves."""
    st, err = attend_call(T=1 << 20, B=1 << 20, max_len=1, **ARGS)
    assert st == -1 and "uwc_kv_attend: too many tokens" in err
