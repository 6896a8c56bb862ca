"""The largest 8-bit conversions on the host side, without a GPU: what is not refused has fewer than 2^32 threads along each
axis of its launch, which is as many as a launch can have."""
import pytest

from tests.test_experts_host_side import child  # noqa: F401

CALLS = """
def launch(name, **change):
    log, error = call(name, **change)
    words = [line.split() for line in launches(log)]
    threads = [max(int(w[1]) * int(w[4]), int(w[2]), int(w[3])) for w in words if w[0] == "launch"]
    return threads, error
"""


@pytest.mark.parametrize("name", ["fp8_quantize", "fp8_dequantize"])
@pytest.mark.parametrize("block", [1, 128])
def test_columns(child, name, block):  # noqa: F811
    trans = "trans=NO_TRANS, " if name == "fp8_quantize" else ""
    got = child(CALLS + f"""
print(json.dumps([launch({name!r}, {trans}block={block}, n=2 ** 26 - d, k=300, ldx=300, lds=2 ** 26) for d in range(6)]))
""")
    for d, (threads, error) in enumerate(got):
        if d < 4:
            assert threads == [] and "status -1" in error and "n must be" in error, (d, threads, error)
        else:
            assert error is None and len(threads) == 1 and threads[0] < 2 ** 32, (d, threads, error)


@pytest.mark.parametrize("trans,block", [("TRANS", 1), ("TRANS", 128), ("NO_TRANS", 128)])
def test_blocks_of_128_columns(child, trans, block):  # noqa: F811
    """2^16 blocks of 128 along k."""
    got = child(CALLS + f"""
print(json.dumps([launch("fp8_quantize", trans={trans}, block={block}, n=n, k=2 ** 23, ldx=2 ** 23, ld=2 ** 23, lds=2 ** 15)
                  for n in (2 ** 14, 2 ** 14 - 127, 2 ** 14 - 128)]))
""")
    for threads, error in got[:2]:
        assert threads == [] and "status -1" in error and "blocks" in error, (threads, error)
    assert got[2][1] is None and len(got[2][0]) == 1 and got[2][0][0] < 2 ** 32, got[2]
