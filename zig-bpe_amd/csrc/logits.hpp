// What the context-free operators (logits.hip) share with the entry points of a context (capi.hip).
#pragma once

namespace zbpe {
const char *thread_message();  // of the calling thread's last failed call without a context; null: it has none
void forget_thread_message();
}
