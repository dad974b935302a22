"""The cache in 8 bits where its kernels have to agree with the definition and with each other."""
import dataclasses

import pytest

from test_gpu_q8 import DT, Cache, check, decode, ints, queries

pytestmark = pytest.mark.gpu


# ---- rows that see no key --------------------------------------------------------------------------------------------------

@dataclasses.dataclass
class Rows:
    """A cache as one of its requests sees it."""
    c: Cache
    row: int = 0

    def __getattr__(self, name):
        return self.c.table[self.row:self.row + 1] if name == "table" else getattr(self.c, name)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("tokens,bound", [(40, 300), (12, 2000), (5, 3000), (2, 5000), (1, 20000)])
def test_decode_rows_without_keys_in_clusters(dtype, hd, tokens, bound):
    """Rows that see nothing beside rows that see some, and calls of such rows alone, with contexts in one part, in clusters of every size
    and in ranges of clusters."""
    from kllm_b200 import kernels
    H, G = 8, 8 if tokens > 2 else 1
    starts, lens = [(37 * i) % 300 for i in range(tokens)], [1] * tokens
    c = Cache(starts, lens, G, hd, 16, seed=tokens)
    q = queries(tokens, H, hd, dtype, seed=6)
    for every in (1, 2):
        pos = [-1 - i if i % every == 0 else s for i, s in enumerate(starts)]
        for _ in range(3):
            got = decode(c, q, ints(*pos), H, G, hd, bound=bound)
            assert not got[::every].any()
            for i in range(1, tokens, every) if every == 2 else ():
                check(got[i:i + 1], q[i:i + 1], Rows(c, i), [starts[i]], [1], H, G, hd)
    if tokens == 1:
        assert kernels.decode_q8_parts(1, G, H // G, hd, bound)[0] > 1
