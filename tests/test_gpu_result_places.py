"""GPU tests of results that share memory with arguments: refused in front of any launch, where CTAs would read what others have written."""
import numpy as np
import pytest

from tests import drafts_model
from tests.test_gpu_drafts import batch, ints, on_device, outputs

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_results_of_a_verification_over_the_rows(tq, dtype):
    """Over the target's or the draft's rows: refused.  Between rows that are apart, or behind the last: as anywhere."""
    rng = np.random.default_rng(1)
    counts, vocab, pad = [5, 6], 40, 16
    parents, tokens, target, draft, u = batch(rng, counts, vocab, 2, True, dtype)
    args = ints([0, 5, 11]), ints(np.concatenate(parents)), ints(tokens)
    uniforms, es = torch.from_numpy(u).cuda(), np.dtype(dtype).itemsize
    want = [drafts_model.verify(parents[i], tokens[r], target[r], draft[r], u[r], 2) for i, r in enumerate((slice(0, 5), slice(5, 11)))]
    for which in (0, 1):
        rows = [on_device(x, pad) for x in (target, draft)]
        numbers = rows[which].as_strided((11 * (vocab + pad),), (1,)).view(torch.int32)
        row = (vocab + pad) * es // 4      # of whole numbers
        for change in ({"next": numbers[:2]}, {"kept": numbers[vocab * es // 4 - 1:][:2]}, {"path": numbers[10 * row:][:4].view(2, 2)}, {"path": numbers[row - 3:][:4].view(2, 2)},
                       {"next": numbers[4 * row - 1:][:2]}, {"kept": numbers[10 * row + 1:][:2]}):
            with pytest.raises(tq.TQError, match="must not be where"):
                tq.verify_drafts(*args, *rows, uniforms, **{**outputs(2, 2), **change})
        gap = numbers[3 * row + vocab * es // 4:][:pad * es // 4]
        out = {"path": gap[:4].view(2, 2), "kept": gap[4:6], "next": gap[6:8]}
        tq.verify_drafts(*args, *rows, uniforms, **out)
        assert out["next"].tolist() == [t for _, t in want] and out["path"].tolist() == [p + [-1] * (2 - len(p)) for p, _ in want]
        assert torch.equal(rows[which].cpu(), torch.from_numpy((target, draft)[which]))
