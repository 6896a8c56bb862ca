"""Which conversions go past the caches, without a GPU: more than 32 MB of values, and where rows are read along the strided
axis or values are written, only at whole dwords."""
from tests.test_experts_host_side import child  # noqa: F401

CALLS = """
import re

def streams(name, **change):
    log, error = call(name, **change)
    assert error is None, error
    (line,) = [l for l in log if l.startswith("launch")]
    # the last truth value among the kernel's template arguments
    return re.findall("Lb([01])E", line.split()[5])[-1] == "1"
"""


def test_quantising(child):  # noqa: F811
    got = child(CALLS + """
out = []
for trans in (NO_TRANS, TRANS):
    for block in (1, 128):
        for type, X, pad, n in ((BF16, P, 0, 4224), (BF16, P, 1, 4224), (BF16, P + 2, 0, 4224), (F16, P, 2, 4224), (F16, P, 3, 4224),
                                (F32, P, 1, 4224), (BF16, P, 0, 128)):
            out.append(streams("fp8_quantize", type=type, trans=trans, block=block, k=4224, n=n, X=X,
                               ldx=(n if trans == TRANS else 4224) + pad, ld=4224, lds=n))
print(json.dumps(out))
""")
    along = [True, True, True, True, True, True, False]  # only codes are stored past the caches
    strided = [True, False, False, True, False, True, False]
    assert got == along * 2 + strided * 2


def test_dequantising(child):  # noqa: F811
    got = child(CALLS + """
print(json.dumps([streams("fp8_dequantize", type=t, block=1, k=4224, n=n, ld=4224, lds=n, X=X, ldx=4224 + pad)
                  for t, X, pad, n in ((BF16, P, 0, 4224), (BF16, P, 1, 4224), (F16, P + 2, 0, 4224), (F32, P, 1, 4224), (F32, P, 0, 128))]))
""")
    assert got == [True, False, False, True, False]
