"""What a cache's status word is reported as: the code, a text that names the fault, and once only."""
import pytest

from ane import _abi
from test_gpu_pages import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("word,code,text", [(1, _abi.LLM_ERR_DEVICE, "bounded wait expired"), (2, _abi.LLM_ERR_DEVICE, "bad page index"),
                                            (3, _abi.LLM_ERR_OOM, "exhausted"), (4, _abi.LLM_ERR_INVALID, "out of range"),
                                            (5, _abi.LLM_ERR_DEVICE, "unknown")])
def test_status_words(word, code, text):
    c = make(pages=4)
    c.check()
    c.status.fill_(word)
    with pytest.raises(_abi.LLMError) as e:
        c.check()
    assert e.value.code == code and text in str(e.value)
    c.check()
