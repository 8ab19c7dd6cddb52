"""Ways into the 4-bit store besides a prefill, over both records."""
import pytest

import kv4_store_cases as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("record", ["cpu", "cuda"])
@pytest.mark.parametrize("how", ["bulk", "one by one"])
def test_ingested_chunks(cuda, record, how):
    K.check_ingest(cuda, record, how)


@pytest.mark.parametrize("record", ["cpu", "cuda"])
def test_prefill_windows_are_exact(cuda, record):
    K.check_prefill_windows_are_exact(cuda, record)
