"""CPU: what the kernels' inline assembly says of itself to the compiler."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'torch-blocksparse_amd', 'csrc')


def statements():
    """(file, template, all of the statement) of every asm statement of the sources"""
    for path in sorted(glob.glob(os.path.join(CSRC, '*'))):
        text = open(path).read()
        for at in re.finditer(r'\basm\b\s*(?:volatile)?\s*\(', text):
            depth, i, quoted = 1, at.end(), False
            while depth:
                if text[i] == '"' and text[i - 1] != '\\':
                    quoted = not quoted
                elif not quoted:
                    depth += (text[i] == '(') - (text[i] == ')')
                i += 1
            whole = text[at.end():i - 1]
            yield os.path.basename(path), whole.split('" :', 1)[0], whole


def test_m0_is_named_where_it_is_written():
    """The compiler keeps values in m0 of its own (addresses of LDS, lanes): a statement that writes it has to say so."""
    writers = [(path, whole) for path, template, whole in statements() if re.search(r's_\w+ m0\b', template)]
    assert len(writers) >= 4
    assert [path for path, whole in writers if not re.search(r':[^:]*"m0"[^:]*$', whole)] == []
