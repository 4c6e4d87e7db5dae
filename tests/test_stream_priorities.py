"""Every stream keeps the default priority: streams of different priorities working side by side have hung on this part."""
import ast
import pathlib

ROOT = pathlib.Path(__file__).resolve().parents[1]
FOLDERS = ('some_amd', 'tools', 'inference', 'modules', 'utils', 'oracle', 'deployment', 'perf')


def test_no_source_asks_for_another_stream_priority():
    python = [p for f in FOLDERS for p in (ROOT / f).rglob('*.py')] + list(ROOT.glob('*.py'))
    native = [p for f in FOLDERS for x in ('*.hip', '*.cpp', '*.h', '*.sh') for p in (ROOT / f).rglob(x)]
    assert len(python) > 30 and len(native) > 10
    found = []
    for p in python:
        for node in ast.walk(ast.parse(p.read_text())):
            if isinstance(node, ast.Call):
                name = node.func.attr if isinstance(node.func, ast.Attribute) else getattr(node.func, 'id', '')
                for kw in node.keywords:
                    if kw.arg == 'is_high_priority_stream' or (kw.arg == 'priority' and name in ('Stream', 'ExternalStream')):
                        found.append(f'{p.relative_to(ROOT)}:{node.lineno}')
                if any(isinstance(a, ast.Constant) and isinstance(a.value, str) and 'priority' in a.value for a in node.args) and name == 'add_argument':
                    found.append(f'{p.relative_to(ROOT)}:{node.lineno}')
    for p in native:
        text = p.read_text(errors='replace')
        if 'StreamCreateWithPriority' in text or 'comm-priority' in text:
            found.append(str(p.relative_to(ROOT)))
    assert not found
