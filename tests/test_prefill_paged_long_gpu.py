"""Chunks as long contexts have them: eight panels of new rows and a ragged ninth, and prefixes of 130000 rows.  Reference and
tolerances are those of test_prefill_paged_gpu.py."""
import pytest

from test_prefill_paged_gpu import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,d,page", [(2, 1, 128, 64), (2, 2, 64, 16), (3, 1, 68, 48)])
@pytest.mark.parametrize("lens,counts", [([3000], [2048]), ([777, 40], [2100, 1300])], ids=str)
def test_many_panels(lens, counts, Hq, Hkv, d, page):
    print(f"case {lens} {counts} {Hq}/{Hkv} d={d} page={page}", flush=True)
    run(make(lens, counts, Hq, Hkv, d, page))


@pytest.mark.parametrize("Hq,Hkv,d,page", [(4, 1, 128, 256), (2, 1, 64, 64), (1, 1, 96, 100)])
@pytest.mark.parametrize("count", [1, 300])
def test_long_prefixes(count, Hq, Hkv, d, page):
    print(f"case 130000 + {count} {Hq}/{Hkv} d={d} page={page}", flush=True)
    run(make([130000], [count], Hq, Hkv, d, page))
